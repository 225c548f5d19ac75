"""The paged 8-bit KV cache in numpy, in 64 bits, from its definition in
include/vxh.h, and ctypes bindings for its entry points."""
import ctypes as C

import numpy as np

import _native as N

INT8, E4M3 = 1, 2
TOP = {INT8: 127.0, E4M3: 448.0}


class Kvq(C.Structure):
    _fields_ = [("type", C.c_int), ("page", C.c_int), ("n_pages", C.c_int), ("n_kv_heads", C.c_int),
                ("head_dim", C.c_int), ("k", C.c_void_p), ("v", C.c_void_p), ("ks", C.c_void_p), ("vs", C.c_void_p)]


class Workspace(C.Structure):
    _fields_ = [("acc", C.c_void_p), ("acc_elems", C.c_size_t), ("part", C.c_void_p), ("part_floats", C.c_size_t)]


def bind(L):
    vp, i, z = C.c_void_p, C.c_int, C.c_size_t
    L.vxh_kvq_alloc.argtypes = [vp, i, i, i, i, i]
    L.vxh_kvq_free.argtypes = [vp]
    L.vxh_page_tables.argtypes = [vp, vp, i, i, vp, i, vp, i, vp, vp, vp, vp, i, vp, vp]
    L.vxh_kvq_write.argtypes = [vp, vp, i, vp, i, vp, i, vp]
    L.vxh_kvq_read.argtypes = [vp, vp, i, vp, i, vp, i, vp]
    L.vxh_attention_kvq.argtypes = [vp, i, vp, vp, i, i, i, vp, i, i, vp, i, vp, i, vp, vp]
    L.vxh_attention_kvq_workspace_floats.argtypes = [i, i, i, i, i]
    L.vxh_attention_kvq_workspace_floats.restype = z
    L.vxh_workspace_alloc.argtypes = [vp, z, z]
    L.vxh_workspace_free.argtypes = [vp]
    L.vxh_capture_begin.argtypes = [vp]
    L.vxh_capture_end.argtypes = [vp, vp]
    L.vxh_graph_launch.argtypes = [vp, vp]
    L.vxh_graph_destroy.argtypes = [vp]
    return L


# --------------------------------------------------------------------------
# codes
# --------------------------------------------------------------------------
def e4m3_table():
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v[(b & 127) == 127] = np.nan
    return np.where(b & 128, -v, v)


E4M3_VALUES = e4m3_table()


def nearest(y, kind):
    """Values of the codes nearest to y (64 bits), ties to even, saturating."""
    if kind == INT8:
        return np.clip(np.rint(y), -127, 127)
    a = np.abs(y)
    e = np.floor(np.log2(np.maximum(a, 2.0 ** -20)))
    e = e + (a >= 2.0 ** (e + 1)) - (a < 2.0 ** e)
    step = 2.0 ** (np.maximum(e, -6) - 3)
    return np.clip(np.rint(y / step) * step, -448, 448)


class Cache:
    """codes (as values) [page][kv head][token][dim] and fp32 scales, written
    as vxh_kvq_write says."""

    def __init__(self, kind, page, n_pages, kv, hd):
        self.kind, self.page, self.n_pages, self.kv, self.hd = kind, page, n_pages, kv, hd
        self.code = [np.zeros((n_pages, kv, page, hd)) for _ in range(2)]
        self.scale = [np.zeros((n_pages, kv), np.float32) for _ in range(2)]

    def write(self, k, v, slot):
        top = np.float32(TOP[self.kind])
        by_page = {}
        for r, s in enumerate(slot):
            if 0 <= s < self.n_pages * self.page:
                by_page.setdefault(int(s) // self.page, {}).setdefault(int(s) % self.page, []).append(r)
        for w, rows in enumerate((k, v)):
            x = np.asarray(rows, np.float32).reshape(len(slot), self.kv, self.hd)
            for p, offs in by_page.items():
                # of two rows of one slot the later one counts, for the scale too
                last = {o: rr[-1] for o, rr in offs.items()}
                new = x[list(last.values())]
                fin = np.where(np.isfinite(new), np.abs(new), np.float32(0))
                amax = fin.max(axis=(0, 2))
                fit = np.where(amax >= np.float32(2.0 ** -100), amax / top, np.float32(0)).astype(np.float32)
                old = np.zeros(self.kv, np.float32) if 0 in last else self.scale[w][p]
                sc = np.maximum(old, fit)
                div = np.where(sc > 0, sc, 1).astype(np.float64)[:, None, None]
                grown = sc > old
                if 0 not in last:
                    again = nearest(self.code[w][p] * old.astype(np.float64)[:, None, None] / div, self.kind)
                    self.code[w][p] = np.where(grown[:, None, None], again, self.code[w][p])
                with np.errstate(invalid="ignore"):
                    y = np.where(np.isnan(new), 0, np.clip(new.astype(np.float64), -1e39, 1e39)).transpose(1, 0, 2)
                y = np.where((sc > 0)[:, None, None], y / div, 0)
                self.code[w][p][:, list(last.keys())] = nearest(y, self.kind)
                self.scale[w][p] = sc

    def values(self, w, slots):
        s = np.asarray(slots)
        p, o = s // self.page, s % self.page
        c = self.code[w][p, :, o].astype(np.float32)
        return (c * self.scale[w][p][:, :, None]).reshape(len(s), -1)


def tables(len_, add, page, free, table, max_rows):
    """vxh_page_tables in plain loops: (table, len_out, row0, pos, slot, counts)."""
    table = table.copy()
    n, a = np.maximum(len_, 0).astype(np.int64), np.maximum(add, 0).astype(np.int64)
    have, need = -(-n // page), -(-(n + a) // page)
    rows, pages = int(a.sum()), int((need - have).sum())
    flag = (pages > len(free)) + 2 * (rows > max_rows) + 4 * bool((need > table.shape[1]).any())
    row0 = np.zeros(len(n) + 1, np.int32)
    pos, slot = np.full(max_rows, -1, np.int32), np.full(max_rows, -1, np.int32)
    if flag:
        return table, n.astype(np.int32), row0, pos, slot, np.array([0, 0, flag, pages])
    it = r = 0
    for b in range(len(n)):
        for j in range(have[b], need[b]):
            table[b, j] = free[it]
            it += 1
        row0[b + 1] = row0[b] + a[b]
        for i in range(a[b]):
            pos[r] = n[b] + i
            slot[r] = table[b, pos[r] // page] * page + pos[r] % page
            r += 1
    return table, (n + a).astype(np.int32), row0, pos, slot, np.array([rows, pages, 0, pages])


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------
def attend(q, cache, row0, len_, table, n_heads, cap, out):
    """The definition in 64 bits; returns (rows, tolerance per row).

    Tolerance, for operands kept to 22 bits (two fp16 parts, each product
    exact in fp32) and fp32 sums: a score is off by at most
    (2^-21 + hd 2^-24) A, A = max_t sum |q K_t|/sqrt(hd) (22-bit operands; every
    partial sum of hd terms rounded once), its place in the exponential by
    2^-23 |score| <= 2^-23 A more, twice (score and maximum); exp, the product's
    two parts and the sums over tokens add 2^-20.  A relative error e of every
    p moves sum p V / sum p by at most 2 e max |V|."""
    hd, kv, page = cache.hd, cache.kv, cache.page
    G = n_heads // kv
    out = out.astype(np.float64)
    tol = np.zeros(out.shape[0])
    for b in range(len(len_)):
        m, n = row0[b + 1] - row0[b], min(int(len_[b]), table.shape[1] * page)
        cols = table[b, :-(-max(n, 0) // page)]
        good = (cols >= 0) & (cols < cache.n_pages)
        use = np.where(good, cols, 0)
        K = (cache.code[0][use] * cache.scale[0][use].astype(np.float64)[:, :, None, None])
        V = (cache.code[1][use] * cache.scale[1][use].astype(np.float64)[:, :, None, None])
        K = K.transpose(1, 0, 2, 3).reshape(kv, -1, hd)
        V = V.transpose(1, 0, 2, 3).reshape(kv, -1, hd)
        live = np.repeat(good, page)
        for i in range(m):
            r = row0[b] + i
            end = n - m + i + 1
            if cap:
                end = min(end, cap)
            out[r, :n_heads * hd] = 0
            ok = np.flatnonzero(live[:max(end, 0)])
            for h in range(n_heads):
                if not len(ok):
                    continue
                qr = q[r, h * hd:(h + 1) * hd].astype(np.float64)
                kk, vv = K[h // G][ok], V[h // G][ok]
                s = kk @ qr / np.sqrt(hd)
                p = np.exp(s - s.max())
                out[r, h * hd:(h + 1) * hd] = p @ vv / p.sum()
                A = (np.abs(kk) @ np.abs(qr)).max() / np.sqrt(hd)
                e = 2 * ((2.0 ** -21 + hd * 2.0 ** -24) + 2.0 ** -23) * A + 2.0 ** -20
                tol[r] = max(tol[r], 2 * e * np.abs(vv).max())
    return out, tol


# --------------------------------------------------------------------------
# device side
# --------------------------------------------------------------------------
class DevCache:
    def __init__(self, L, kind, page, n_pages, kv, hd):
        self.L, self.s = L, Kvq()
        self.ref = C.byref(self.s)
        rc = L.vxh_kvq_alloc(self.ref, kind, page, n_pages, kv, hd)
        assert rc == 0, L.vxh_last_error()
        self.kind, self.page, self.n_pages, self.kv, self.hd = kind, page, n_pages, kv, hd

    def read(self, slots, fill=-7.0):
        s = np.asarray(slots, np.int32)
        w = self.kv * self.hd
        ds, dk, dv = (N.DevBuf(self.L, a) for a in (s, np.full((len(s), w), fill, np.float32),
                                                    np.full((len(s), w), fill, np.float32)))
        assert self.L.vxh_kvq_read(self.ref, ds.ptr, len(s), dk.ptr, w, dv.ptr, w, None) == 0, self.L.vxh_last_error()
        out = [d.get(np.float32, len(s) * w).reshape(len(s), w) for d in (dk, dv)]
        for d in (ds, dk, dv):
            d.free()
        return out

    def scales(self):
        n = self.n_pages * self.kv
        out = []
        for p in (self.s.ks, self.s.vs):
            a = np.zeros(n, np.float32)
            assert self.L.vxh_download(N._ptr(a), C.c_void_p(p), a.nbytes, None) == 0
            out.append(a.reshape(self.n_pages, self.kv))
        return out

    def write(self, k, v, slot, ldk=None, ldv=None, stream=None):
        s = np.asarray(slot, np.int32)
        w = self.kv * self.hd
        ldk, ldv = ldk or w, ldv or w
        kk, vv = np.full((len(s), ldk), np.nan, np.float32), np.full((len(s), ldv), np.nan, np.float32)
        kk[:, :w], vv[:, :w] = k, v
        bufs = [N.DevBuf(self.L, a) for a in (kk, vv, s)]
        rc = self.L.vxh_kvq_write(self.ref, bufs[0].ptr, ldk, bufs[1].ptr, ldv, bufs[2].ptr, len(s), stream)
        assert rc == 0, self.L.vxh_last_error()
        assert self.L.vxh_stream_sync(stream) == 0
        for b in bufs:
            b.free()

    def bytes(self):
        n = self.n_pages * self.kv * self.page * self.hd
        out = []
        for p in (self.s.k, self.s.v):
            a = np.zeros(n, np.uint8)
            assert self.L.vxh_download(N._ptr(a), C.c_void_p(p), a.nbytes, None) == 0
            out.append(a.reshape(self.n_pages, self.kv, -1))
        return out

    def put(self, which, page, head, raw):
        """Raw bytes of one page and head of K (0) or V (1)."""
        raw = np.ascontiguousarray(raw, np.uint8)
        at = (self.s.k, self.s.v)[which] + (int(page) * self.kv + head) * self.page * self.hd
        assert self.L.vxh_upload(C.c_void_p(at), N._ptr(raw), raw.nbytes, None) == 0

    def put_scale(self, which, page, head, value):
        a = np.array([value], np.float32)
        at = (self.s.ks, self.s.vs)[which] + 4 * (int(page) * self.kv + head)
        assert self.L.vxh_upload(C.c_void_p(at), N._ptr(a), 4, None) == 0

    def free(self):
        assert self.L.vxh_kvq_free(self.ref) == 0


def run_attend(L, dc, q, row0, len_, table, n_heads, cap, max_rows=None, max_seq_rows=None, ld_extra=0, out_extra=0,
               stream=None, fill=-3.0):
    """vxh_attention_kvq on fresh buffers; returns out[max_rows][n_heads * hd]."""
    w = n_heads * dc.hd
    R = max_rows or q.shape[0]
    ldq, ldo = w + ld_extra, w + out_extra
    qq = np.full((R, ldq), np.nan, np.float32)
    qq[:q.shape[0], :w] = q
    m = int(max(np.diff(row0).max(), 1)) if max_seq_rows is None else max_seq_rows
    bufs = [N.DevBuf(L, a) for a in (qq, np.asarray(row0, np.int32), np.asarray(len_, np.int32),
                                     np.ascontiguousarray(table, np.int32), np.full((R, ldo), fill, np.float32))]
    ws = Workspace()
    n = L.vxh_attention_kvq_workspace_floats(R, len(len_), n_heads, dc.kv, dc.hd)
    assert L.vxh_workspace_alloc(C.byref(ws), 32, n) == 0
    rc = L.vxh_attention_kvq(bufs[0].ptr, ldq, bufs[1].ptr, bufs[2].ptr, len(len_), R, m, bufs[3].ptr, table.shape[1],
                             n_heads, dc.ref, cap, bufs[4].ptr, ldo, C.byref(ws), stream)
    assert rc == 0, L.vxh_last_error()
    assert L.vxh_stream_sync(stream) == 0
    out = bufs[4].get(np.float32, R * ldo).reshape(R, ldo)
    assert np.all(out[:, w:] == fill), "columns past the heads were written"
    for b in bufs:
        b.free()
    L.vxh_workspace_free(C.byref(ws))
    return out[:, :w]
