"""The paged 8-bit KV cache as measurable cases: page tables and slot maps of a
serving step, the write of new rows into the cache (and their read-back), and
the attention of a ragged batch over it.

Shapes are those of the repository's configurations (a 22-layer draft with 32/4
heads of 64, a 7B-shape target with 32/32 heads of 128, a GQA model with 28/4
heads of 128) at serving batches around them.

A cache is held here in its logical form, codes[page][kv head][token][dim]
(int8, or e4m3 as its bytes) with scales[page][kv head]; where the framework's
kernels run it is laid out as include/vxh.h says.
"""
import ctypes as C
import os

import torch

own = False

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(os.path.dirname(HERE), "veltrix-engine_amd", "lib", "libveltrix_amd.so")
DEV = "cuda"
vp = C.c_void_p

TYPES = {"int8": (1, 127.0), "e4m3": (2, 448.0)}
TINY = 2.0 ** -100      # blocks whose largest value is below this are zeros


# --------------------------------------------------------------------------
# the library
# --------------------------------------------------------------------------
class Kvq(C.Structure):
    _fields_ = [("type", C.c_int), ("page", C.c_int), ("n_pages", C.c_int), ("n_kv_heads", C.c_int),
                ("head_dim", C.c_int), ("k", vp), ("v", vp), ("ks", vp), ("vs", vp)]


class Workspace(C.Structure):
    _fields_ = [("acc", vp), ("acc_elems", C.c_size_t), ("part", vp), ("part_floats", C.c_size_t)]


_lib = None


def lib():
    global _lib
    if _lib is None:
        torch.zeros(1, device=DEV)
        L = C.CDLL(LIB)
        i, z = C.c_int, C.c_size_t
        L.vxh_kvq_alloc.argtypes = [vp, i, i, i, i, i]
        L.vxh_kvq_free.argtypes = [vp]
        L.vxh_workspace_alloc.argtypes = [vp, z, z]
        L.vxh_workspace_free.argtypes = [vp]
        L.vxh_page_tables.argtypes = [vp, vp, i, i, vp, i, vp, i, vp, vp, vp, vp, i, vp, vp]
        L.vxh_kvq_write.argtypes = [vp, vp, i, vp, i, vp, i, vp]
        L.vxh_kvq_read.argtypes = [vp, vp, i, vp, i, vp, i, vp]
        L.vxh_attention_kvq.argtypes = [vp, i, vp, vp, i, i, i, vp, i, i, vp, i, vp, i, vp, vp]
        L.vxh_attention_kvq_workspace_floats.argtypes = [i, i, i, i, i]
        L.vxh_attention_kvq_workspace_floats.restype = z
        L.vxh_last_error.restype = C.c_char_p
        if L.vxh_init() != 0:
            raise RuntimeError(L.vxh_last_error().decode())
        _lib = L
    return _lib


def ok(rc):
    if rc != 0:
        raise RuntimeError("%d: %s" % (rc, _lib.vxh_last_error().decode()))


def ptr(t):
    return vp(t.data_ptr())


def stream():
    return vp(torch.cuda.current_stream().cuda_stream)


class Owned:
    """A struct the library fills, given back when the state goes."""

    def __init__(self, struct, free):
        self.s, self.free = struct, free
        self.ref = C.byref(struct)

    def __del__(self):
        self.free(self.ref)


class DeviceBytes:
    """Library memory as an array (for filling a cache)."""

    def __init__(self, owner, address, n, typestr="|u1"):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": (n,), "typestr": typestr, "data": (address, False), "version": 2}


def packed_k(codes):
    """codes[page][head][token][dim] bytes in the cache's order: 32 tokens and
    32 dims at a time, lane 16 g + n holding dims 8 g.. of tokens n and n + 16."""
    p, h, t, d = codes.shape
    x = codes.view(p, h, t // 32, 2, 16, d // 32, 4, 8)        # page head T half n J g e
    return x.permute(0, 1, 2, 5, 6, 4, 3, 7).reshape(-1)


def packed_v(codes):
    """The same for values: lane 16 g + n holds dims n and n + 16 of tokens
    4 g.. and 16 + 4 g.."""
    p, h, t, d = codes.shape
    x = codes.view(p, h, t // 32, 2, 4, 4, d // 32, 2, 16)     # page head T half g i J hh n
    return x.permute(0, 1, 2, 6, 4, 8, 7, 3, 5).reshape(-1)


def stored(codes, kind):
    """A code's byte in the cache: int8 with an offset of 128, e4m3 as it is."""
    return (codes.to(torch.int16) + 128).to(torch.uint8) if kind == "int8" else codes


def make_cache(case, k, v, ks, vs):
    """The framework's cache with the logical contents k, v, ks, vs."""
    L = lib()
    c = Owned(Kvq(), L.vxh_kvq_free)
    n_pages, kv, page, hd = k.shape
    ok(L.vxh_kvq_alloc(c.ref, TYPES[case["type"]][0], page, n_pages, kv, hd))
    for address, codes, pack in ((c.s.k, k, packed_k), (c.s.v, v, packed_v)):
        dst = torch.as_tensor(DeviceBytes(c, address, codes.numel()), device=DEV)
        step = max(1, (1 << 28) // codes[0].numel())
        for p in range(0, n_pages, step):
            part = pack(stored(codes[p:p + step], case["type"]))
            dst[p * codes[0].numel():p * codes[0].numel() + part.numel()] = part
    for address, scale in ((c.s.ks, ks), (c.s.vs, vs)):
        torch.as_tensor(DeviceBytes(c, address, scale.numel(), "<f4"), device=DEV).copy_(scale.reshape(-1))
    torch.cuda.synchronize()
    return c


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
class State:
    pass


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def pages_of(n, page):
    return -(-n // page)


def lengths(case):
    """Tokens cached before the step and rows added by it, one pair a request.
    "ragged" requests lie anywhere between none and the longest."""
    n, past, rows = case["seqs"], case["past"], case["rows"]
    g = torch.Generator().manual_seed(1000 * n + past)
    if case["ragged"]:
        lens = [int(x) for x in torch.randint(0, past + 1, (n,), generator=g)]
        lens[-1] = past
    else:
        lens = [past] * n
    adds = [rows] * n
    for i in range(case.get("prompts", 0)):      # some requests bring a prompt chunk instead
        adds[(i * 7) % n] = case["chunk"]
    return lens, adds


def random_codes(g, kind, n_pages, kv, page, hd):
    """Codes as a normal distribution leaves them, and scales within a factor of four."""
    out = torch.empty(n_pages, kv, page, hd, dtype=torch.int8 if kind == "int8" else torch.uint8, device=DEV)
    step = max(1, (1 << 26) // (kv * page * hd))
    for p in range(0, n_pages, step):
        x = normal(g, min(step, n_pages - p), kv, page, hd)
        if kind == "int8":
            out[p:p + step] = torch.clamp(torch.round(x * 34), -127, 127).to(torch.int8)
        else:
            out[p:p + step] = torch.clamp(x * 120, -448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    s = (0.03 if kind == "int8" else 0.008) * 2.0 ** (2 * torch.rand(n_pages, kv, generator=g, device=DEV) - 1)
    return out, s


def values(codes, kind):
    return codes.float() if kind == "int8" else codes.view(torch.float8_e4m3fn).float()


def page_plan(case, seed, lens, adds):
    """A pool whose pages lie in random order: table[request][column]."""
    page = case["page"]
    need = [pages_of(n + a, page) for n, a in zip(lens, adds)]
    pool = sum(need) + 3
    g = torch.Generator().manual_seed(seed + 77)
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    cols = max(max(need), 1)
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, pool


def row_starts(adds):
    out = [0]
    for a in adds:
        out.append(out[-1] + a)
    return out


# --------------------------------------------------------------------------
# tables: page tables, row positions and slots of one step
# --------------------------------------------------------------------------
def prepare_tables(case, seed):
    s = State()
    lens, adds = lengths(case)
    page = case["page"]
    table, pool = page_plan(case, seed, lens, [0] * len(lens))
    fresh = [pages_of(n + a, page) - pages_of(n, page) for n, a in zip(lens, adds)]
    cols = max(pages_of(n + a, page) for n, a in zip(lens, adds)) + 1
    s.table = torch.full((len(lens), cols), -1, dtype=torch.int32, device=DEV)
    s.table[:, :table.shape[1]] = table.to(DEV)[:, :cols]
    n_free = max(1, sum(fresh) + (5 if not case["short"] else -1))
    g = gen(seed)
    s.free = (torch.randperm(n_free, generator=g, device=DEV) + pool).to(torch.int32)
    s.len, s.add = ints(lens), ints(adds)
    s.page, s.n, s.max_rows = page, len(lens), sum(adds) + 7
    if own:
        L = lib()
        s.call = L.vxh_page_tables
        s.len_out, s.row0 = torch.zeros_like(s.len), torch.zeros(s.n + 1, dtype=torch.int32, device=DEV)
        s.pos, s.slot = (torch.zeros(s.max_rows, dtype=torch.int32, device=DEV) for _ in range(2))
        s.counts = torch.zeros(4, dtype=torch.int32, device=DEV)
        s.args = (ptr(s.len), ptr(s.add), s.n, page, ptr(s.free), n_free, ptr(s.table), cols, ptr(s.len_out),
                  ptr(s.row0), ptr(s.pos), ptr(s.slot), s.max_rows, ptr(s.counts))
    return s


def run_tables(s):
    if own:
        ok(s.call(*s.args, stream()))
        return [s.table, s.len_out, s.row0, s.pos, s.slot, s.counts]
    n, a, page = s.len.long(), s.add.long(), s.page
    have, need = (n + page - 1) // page, (n + a + page - 1) // page
    off = torch.cumsum(need - have, 0) - (need - have)
    row0 = torch.zeros(s.n + 1, dtype=torch.long, device=DEV)
    row0[1:] = torch.cumsum(a, 0)
    taken = (need - have).sum()
    flag = ((taken > s.free.numel()).long() + 2 * (row0[-1] > s.max_rows).long() +
            4 * (need.max() > s.table.shape[1]).long())
    good = flag == 0
    col = torch.arange(s.table.shape[1], device=DEV)[None, :]
    src = torch.clamp(off[:, None] + col - have[:, None], 0, s.free.numel() - 1)
    fresh = (col >= have[:, None]) & (col < need[:, None]) & good
    table = torch.where(fresh, s.free[src], s.table)
    r = torch.arange(s.max_rows, device=DEV)
    b = torch.clamp((r[:, None] >= row0[None, 1:]).sum(1), max=s.n - 1) if s.n * s.max_rows < 1 << 24 else \
        torch.clamp(torch.searchsorted(row0[1:].contiguous(), r, right=True), max=s.n - 1)
    live = (r < row0[-1]) & good
    pos = torch.where(live, n[b] + r - row0[b], -1)
    c = torch.clamp(pos // page, 0, s.table.shape[1] - 1)
    slot = torch.where(live, table[b, c].long() * page + pos % page, -1)
    counts = torch.stack([row0[-1] * good, taken * good, flag, taken])
    return [table, (n + a * good).int(), (row0 * good).int(), pos.int(), slot.int(), counts.int()]


def work_tables(c):
    lens, adds = lengths(c)
    rows = sum(adds)
    fresh = sum(pages_of(n + a, c["page"]) - pages_of(n, c["page"]) for n, a in zip(lens, adds))
    return {"bytes": 16 * c["seqs"] + 8 * rows + 8 * fresh, "flops": 4 * c["seqs"] + 4 * rows}


# --------------------------------------------------------------------------
# write: new rows into the cache, and the tokens of the touched pages read back
# --------------------------------------------------------------------------
def write_inputs(case, seed):
    lens, adds = lengths(case)
    page, kv, hd = case["page"], case["kv_heads"], case["hd"]
    table, pool = page_plan(case, seed, lens, adds)
    slot, back = [], []
    for b, (n, a) in enumerate(zip(lens, adds)):
        at = torch.arange(n, n + a)
        slot.append(table[b][at // page].long() * page + at % page)
        if a:
            at = torch.arange(n // page * page, n + a)
            back.append(table[b][at // page].long() * page + at % page)
    slot, back = torch.cat(slot).to(torch.int32).to(DEV), torch.cat(back).to(torch.int32).to(DEV)
    g = gen(seed)
    rows = slot.numel()
    # a few channels of the keys are larger, as rotated keys have them
    gain = 1 + 7 * (torch.rand(kv * hd, generator=g, device=DEV) < 0.03).float()
    k, v = normal(g, rows, kv * hd) * gain, normal(g, rows, kv * hd)
    cache = []
    for _ in range(2):
        cache += random_codes(g, case["type"], pool, kv, page, hd)
    return k, v, slot, back, cache


def prepare_write(case, seed):
    s = State()
    k, v, slot, back, cache = write_inputs(case, seed)
    s.k, s.v, s.slot, s.back, s.case = k, v, slot, back, case
    n, w = back.numel(), k.shape[1]
    if own:
        L = lib()
        kc, ks, vc, vs = cache
        s.cache = make_cache(case, kc, vc, ks, vs)
        s.k_out, s.v_out = torch.zeros(n, w, device=DEV), torch.zeros(n, w, device=DEV)
        s.write, s.read = L.vxh_kvq_write, L.vxh_kvq_read
        s.a0 = (s.cache.ref, ptr(k), w, ptr(v), w, ptr(slot), slot.numel())
        s.a1 = (s.cache.ref, ptr(back), n, ptr(s.k_out), w, ptr(s.v_out), w)
    else:
        s.cache = cache
    return s


def nearest(y, kind):
    """The code values nearest to y (64 bits), ties to even, saturating."""
    if kind == "int8":
        return torch.clamp(torch.round(y), -127, 127)
    e = torch.floor(torch.log2(torch.clamp(y.abs(), min=2.0 ** -20)))
    e = e + (y.abs() >= 2.0 ** (e + 1)).double() - (y.abs() < 2.0 ** e).double()
    step = 2.0 ** (torch.clamp(e, min=-6) - 3)
    return torch.clamp(torch.round(y / step) * step, -448, 448)


def encode(y, kind):
    return y.to(torch.int8) if kind == "int8" else y.float().to(torch.float8_e4m3fn).view(torch.uint8)


def run_write(s):
    if own:
        st = stream()
        ok(s.write(*s.a0, st))
        ok(s.read(*s.a1, st))
        return [s.k_out, s.v_out]
    case = s.case
    kind, page, kv, hd = case["type"], case["page"], case["kv_heads"], case["hd"]
    qmax = TYPES[kind][1]
    pg, off = (s.slot // page).long(), (s.slot % page).long()
    touched, index = torch.unique(pg, return_inverse=True)
    first = torch.zeros(touched.numel(), device=DEV).index_reduce_(0, index, (off == 0).float(), "amax") > 0
    out = []
    for rows, (codes, scales) in ((s.k, s.cache[:2]), (s.v, s.cache[2:])):
        x = rows.view(-1, kv, hd)
        finite = torch.isfinite(x)
        amax = torch.zeros(touched.numel(), kv, device=DEV).index_reduce_(
            0, index, torch.where(finite, x.abs(), 0.0).amax(2), "amax")
        fresh = torch.where(amax >= TINY, (amax.double() / qmax).float(), 0.0)
        old = torch.where(first[:, None], 0.0, scales[touched])
        new = torch.maximum(old, fresh)
        # the tokens that were there, at the new scale
        ratio = torch.where(new > 0, old.double(), 0.0)
        was = values(codes[touched], kind).double()
        was = nearest(was * ratio[:, :, None, None] / torch.where(new > 0, new, 1.0).double()[:, :, None, None], kind)
        keep = (new == scales[touched])[:, :, None, None]
        codes[touched] = torch.where(keep, codes[touched], encode(was, kind))
        scales[touched] = new
        sc = new[index].double()[:, :, None]
        y = torch.where(torch.isnan(x), 0.0, torch.clamp(x, -3e38, 3e38)).double() / torch.where(sc > 0, sc, 1.0)
        codes[pg, :, off] = encode(nearest(torch.where(sc > 0, y, 0.0), kind), kind)
        b_pg, b_off = (s.back // page).long(), (s.back % page).long()
        out.append((values(codes[b_pg, :, b_off], kind) * scales[b_pg][:, :, None]).reshape(s.back.numel(), -1))
    return out


def exact_write(case, seed):
    """Page by page from the definition, in 64 bits."""
    k, v, slot, back, cache = write_inputs(case, seed)
    if slot.numel() > 4096:
        return None
    kind, page, kv, hd = case["type"], case["page"], case["kv_heads"], case["hd"]
    qmax = TYPES[kind][1]
    sl, bk = slot.tolist(), back.tolist()
    by_page = {}
    for r, x in enumerate(sl):
        by_page.setdefault(x // page, []).append((x % page, r))
    outs = []
    for rows, codes, scales in ((k, cache[0], cache[1]), (v, cache[2], cache[3])):
        vals, rows = {}, rows.double().view(-1, kv, hd)
        for p, items in by_page.items():
            offs, rr = [o for o, _ in items], [r for _, r in items]
            new = rows[rr]
            s_old = scales[p].double() if 0 not in offs else torch.zeros(kv, dtype=torch.float64, device=DEV)
            # the scale is held in 32 bits
            s_new = torch.maximum(s_old, (new.abs().amax(dim=(0, 2)) / qmax).float().double())
            div = torch.where(s_new > 0, s_new, 1.0)[:, None, None]
            old = values(codes[p], kind).double()
            old = torch.where((s_new > s_old)[:, None, None], nearest(old * s_old[:, None, None] / div, kind), old)
            old[:, offs] = nearest(new.transpose(0, 1) / div, kind)
            vals[p] = old * s_new[:, None, None]
        outs.append(torch.stack([vals[x // page][:, x % page] for x in bk]).reshape(len(bk), -1))
    return outs


def work_write(c):
    lens, adds = lengths(c)
    rows = sum(adds)
    back = sum(n % c["page"] + a for n, a in zip(lens, adds) if a)
    w = 2 * c["kv_heads"] * c["hd"]
    return {"bytes": rows * w * 5 + back * w * 5 + 4 * (rows + back), "flops": 2 * w * (rows + back)}


# --------------------------------------------------------------------------
# attend: the rows of a ragged batch over the paged cache
# --------------------------------------------------------------------------
def attend_inputs(case, seed):
    lens, adds = lengths(case)
    table, pool = page_plan(case, seed, lens, adds)
    g = gen(seed)
    q = 2 * normal(g, sum(adds), case["heads"] * case["hd"])
    cache = []
    for _ in range(2):
        cache += random_codes(g, case["type"], pool, case["kv_heads"], case["page"], case["hd"])
    return q, [n + a for n, a in zip(lens, adds)], adds, table.to(DEV), cache


def prepare_attend(case, seed):
    s = State()
    q, total, adds, table, cache = attend_inputs(case, seed)
    s.q, s.table, s.case, s.total, s.adds = q, table, case, total, adds
    H, KV, hd = case["heads"], case["kv_heads"], case["hd"]
    if own:
        L = lib()
        kc, ks, vc, vs = cache
        s.cache = make_cache(case, kc, vc, ks, vs)
        s.out = torch.zeros_like(q)
        s.row0, s.len = ints(row_starts(adds)), ints(total)
        R, B = q.shape[0], len(adds)
        s.ws = Owned(Workspace(), L.vxh_workspace_free)
        ok(L.vxh_workspace_alloc(s.ws.ref, 32, L.vxh_attention_kvq_workspace_floats(R, B, H, KV, hd)))
        s.call = L.vxh_attention_kvq
        s.args = (ptr(q), H * hd, ptr(s.row0), ptr(s.len), B, R, max(adds), ptr(table), table.shape[1], H, s.cache.ref,
                  case["cap"], ptr(s.out), H * hd, s.ws.ref)
    else:
        s.cache = cache
    return s


def run_attend(s):
    if own:
        ok(s.call(*s.args, stream()))
        return s.out
    case = s.case
    kind, page, KV, hd, H = case["type"], case["page"], case["kv_heads"], case["hd"], case["heads"]
    G, cap = H // KV, case["cap"] or 1 << 30
    out = torch.empty_like(s.q)
    kc, ks, vc, vs = s.cache
    r = 0
    for b, (n, a) in enumerate(zip(s.total, s.adds)):
        if not a:
            continue
        t = s.table[b, :pages_of(n, page)].long()
        k = (values(kc[t], kind) * ks[t][:, :, None, None]).transpose(0, 1).reshape(KV, -1, hd)[:, :n]
        v = (values(vc[t], kind) * vs[t][:, :, None, None]).transpose(0, 1).reshape(KV, -1, hd)[:, :n]
        q = s.q[r:r + a].view(a, KV, G, hd).permute(1, 2, 0, 3).reshape(KV, G * a, hd)
        sc = torch.matmul(q, k.transpose(1, 2).contiguous()) / hd ** 0.5
        last = torch.clamp(torch.arange(n - a, n, device=DEV) + 1, max=cap).repeat(G)
        sc = sc.masked_fill(torch.arange(n, device=DEV)[None, :] >= last[:, None], float("-inf"))
        p = torch.exp(sc - sc.amax(2, keepdim=True))
        o = torch.matmul(p, v) / p.sum(2, keepdim=True)
        out[r:r + a] = o.view(KV, G, a, hd).permute(2, 0, 1, 3).reshape(a, -1)
        r += a
    return out


def exact_attend(case, seed):
    """Head by head in 64 bits, over each row's own positions."""
    q, total, adds, table, cache = attend_inputs(case, seed)
    kind, page, KV, hd, H = case["type"], case["page"], case["kv_heads"], case["hd"], case["heads"]
    if sum(n * a for n, a in zip(total, adds)) * H > 1 << 29:
        return None
    G, cap = H // KV, case["cap"] or 1 << 30
    kc, ks, vc, vs = cache
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    r = 0
    for b, (n, a) in enumerate(zip(total, adds)):
        if not a:
            continue
        t = table[b, :pages_of(n, page)].long()
        seen = torch.arange(n, device=DEV)[None, :] < torch.clamp(torch.arange(n - a, n, device=DEV)[:, None] + 1, max=cap)
        for g in range(KV):
            kk = (values(kc[t, g], kind).double() * ks[t, g].double()[:, None, None]).reshape(-1, hd)[:n]
            vv = (values(vc[t, g], kind).double() * vs[t, g].double()[:, None, None]).reshape(-1, hd)[:n]
            for h in range(g * G, (g + 1) * G):
                w = q[r:r + a, h * hd:(h + 1) * hd].double() @ kk.T / float(hd) ** 0.5
                w = torch.where(seen, w, -float("inf"))
                w = torch.exp(w - torch.logsumexp(w, 1, keepdim=True))
                out[r:r + a, h * hd:(h + 1) * hd] = w @ vv
        r += a
    return out


def work_attend(c):
    lens, adds = lengths(c)
    H, KV, hd, cap = c["heads"], c["kv_heads"], c["hd"], c["cap"] or 1 << 30
    b = f = 0
    for n, a in zip(lens, adds):
        if a:
            b += 2 * KV * (min(n + a, cap) * hd + 4 * pages_of(min(n + a, cap), c["page"]))
            f += 4 * H * hd * sum(min(n + i + 1, cap) for i in range(a))
    return {"bytes": b + 8 * sum(adds) * H * hd, "flops": f}


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------
OPS = {
    "tables": (prepare_tables, run_tables, None, work_tables),
    "write": (prepare_write, run_write, exact_write, work_write),
    "attend": (prepare_attend, run_attend, exact_attend, work_attend),
}

DRAFT = {"heads": 32, "kv_heads": 4, "hd": 64}
TARGET = {"heads": 32, "kv_heads": 32, "hd": 128}
GQA = {"heads": 28, "kv_heads": 4, "hd": 128}


def kv(shape):
    return {"kv_heads": shape["kv_heads"], "hd": shape["hd"]}


def listed():
    return [
        # the verify step of one conversation: one request, nine rows
        {"name": "tables_one", "op": "tables", "seqs": 1, "past": 2048, "rows": 9, "ragged": False, "page": 32,
         "short": False},
        # a server's step: 1000 conversations decode and 12 more bring prompt chunks
        {"name": "tables_server", "op": "tables", "seqs": 1012, "past": 8192, "rows": 1, "ragged": True, "page": 32,
         "prompts": 12, "chunk": 512, "short": False},
        # one decoded token of the draft
        dict(kv(DRAFT), name="write_one", op="write", type="int8", page=32, seqs=1, past=2047, rows=1, ragged=False),
        # one decoded token of each of 64 conversations of the GQA model
        dict(kv(GQA), name="write_batch", op="write", type="e4m3", page=64, seqs=64, past=4000, rows=1, ragged=True),
        # a 2048-token prompt of the target behind a short one
        dict(kv(TARGET), name="write_prompt", op="write", type="int8", page=32, seqs=1, past=77, rows=2048,
             ragged=False),
        # one decoded token of the draft at a 2K context: launches and latency
        dict(DRAFT, name="attend_one", op="attend", type="int8", page=32, seqs=1, past=2047, rows=1, ragged=False,
             cap=4096),
        # a verify batch of nine rows of the GQA model over 8K
        dict(GQA, name="attend_verify", op="attend", type="int8", page=64, seqs=1, past=8183, rows=9, ragged=False,
             cap=0),
        # 64 decoding conversations of the GQA model, up to 8K each
        dict(GQA, name="attend_batch", op="attend", type="e4m3", page=32, seqs=64, past=8191, rows=1, ragged=True,
             cap=0),
        # verify batches of sixteen conversations of the target, every head its own keys
        dict(TARGET, name="attend_heads", op="attend", type="int8", page=32, seqs=16, past=2048, rows=9, ragged=True,
             cap=4096),
        # two conversations of 128K tokens: few rows, a long axis
        dict(GQA, name="attend_long", op="attend", type="int8", page=128, seqs=2, past=131071, rows=1, ragged=False,
             cap=0),
        # a 2048-token prompt of the target: the matrix products count
        dict(TARGET, name="attend_prompt", op="attend", type="int8", page=32, seqs=1, past=0, rows=2048, ragged=False,
             cap=4096),
        # 24 decoding conversations of the draft with two prompt chunks among them
        dict(DRAFT, name="attend_mixed", op="attend", type="e4m3", page=64, seqs=26, past=2036, rows=1, ragged=True,
             prompts=2, chunk=500, cap=4096),
    ]


def spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["tables", "write", "write", "attend", "attend", "attend", "attend"])
    page, kind = rng.choice([32, 64, 128]), rng.choice(["int8", "e4m3"])
    if op == "tables":
        c = {"op": op, "seqs": spread(rng, 1, 1000), "past": spread(rng, 1, 8192), "rows": rng.choice([0, 1, 1, 3, 9]),
             "ragged": rng.random() < 0.8, "page": page, "short": rng.random() < 0.15}
        if rng.random() < 0.5:
            c.update(prompts=1 + c["seqs"] // 80, chunk=spread(rng, 17, 512))
        return c
    heads = rng.choice([1, 2, 4, 8, 32])
    hd = rng.choice([32, 64, 64, 96, 128, 128, 128])
    c = {"op": op, "type": kind, "page": page, "kv_heads": heads, "hd": hd, "ragged": rng.random() < 0.7}
    style = rng.choice(["decode", "verify", "prompt", "mixed"])
    c["seqs"] = {"decode": spread(rng, 1, 64), "verify": spread(rng, 1, 16), "prompt": rng.randint(1, 3),
                 "mixed": spread(rng, 2, 32)}[style]
    c["rows"] = {"decode": 1, "verify": rng.randint(2, 16), "prompt": spread(rng, 17, 1500 // c["seqs"]),
                 "mixed": 1}[style]
    c["past"] = spread(rng, 1, {"decode": 8192, "verify": 8192, "prompt": 2000, "mixed": 3000}[style])
    if style == "mixed":
        c.update(prompts=rng.randint(1, 2), chunk=spread(rng, 17, 600))
    if heads == 32 and c["seqs"] * c["past"] > 40000:
        c["seqs"] = max(1, 40000 // c["past"])
    if op == "attend":
        c.update(heads=heads * rng.choice([1, 2, 4, 7, 8] if heads < 8 else [1, 1, 4] if heads < 32 else [1]),
                 cap=rng.choice([0, 0, 4096, 1000]))
        if c["heads"] * hd > 4096:
            c["heads"] = heads
    return c


def prepare(case, seed):
    s = OPS[case["op"]][0](case, seed)
    s.op = case["op"]
    return s


def run(state):
    return OPS[state.op][1](state)


def exact(case, seed):
    make = OPS[case["op"]][2]
    return make(case, seed) if make else None


def work(case):
    return OPS[case["op"]][3](case)
