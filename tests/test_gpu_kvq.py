"""The paged 8-bit KV cache on the GPU: page tables against plain loops, the
write bit for bit against the definition in 64 bits, the attention against 64
bits (tolerance derived in _kvq.attend), and steps of serving with all of them
together, eager and as a replayed graph."""
import ctypes as C

import numpy as np
import pytest

import _kvq as Q
import _native as N

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def P():
    if not N.product_available():
        pytest.fail("product library not built")
    L = Q.bind(N.bind_vxh(N.product()))
    assert L.vxh_init() == 0, L.vxh_last_error()
    return L


# --------------------------------------------------------------------------
# page tables
# --------------------------------------------------------------------------
def run_tables(P, len_, add, page, free, table, max_rows, stream=None):
    arrs = [np.asarray(a, np.int32) for a in (len_, add, free if len(free) else [0], table)]
    B = len(len_)
    arrs += [np.full(n, -9, np.int32) for n in (B, B + 1, max_rows, max_rows, 4)]
    bufs = [N.DevBuf(P, a) for a in arrs]
    d = dict(zip(("len", "add", "free", "table", "len_out", "row0", "pos", "slot", "counts"), bufs))
    rc = P.vxh_page_tables(d["len"].ptr, d["add"].ptr, B, page, d["free"].ptr, len(free), d["table"].ptr,
                           arrs[3].shape[1], d["len_out"].ptr, d["row0"].ptr, d["pos"].ptr, d["slot"].ptr, max_rows,
                           d["counts"].ptr, stream)
    assert rc == 0, P.vxh_last_error()
    assert P.vxh_stream_sync(stream) == 0
    out = [d[n].get(np.int32, a.size).reshape(a.shape)
           for n, a in zip(("table", "len_out", "row0", "pos", "slot", "counts"),
                           [arrs[3], arrs[4], arrs[5], arrs[6], arrs[7], arrs[8]])]
    for b in bufs:
        b.free()
    return out


def same_tables(P, len_, add, page, free, table, max_rows):
    got = run_tables(P, len_, add, page, free, table, max_rows)
    want = Q.tables(np.asarray(len_), np.asarray(add), page, free, table, max_rows)
    for name, g, w in zip(("table", "len_out", "row0", "pos", "slot", "counts"), got, want):
        assert np.array_equal(g, w), name
    return got


@pytest.mark.parametrize("B,page,most,rows", [(1, 32, 100, 9), (1, 128, 1, 1), (7, 64, 300, 40), (64, 32, 2000, 1),
                                              (255, 32, 90, 3), (257, 128, 700, 5), (1000, 64, 3000, 2),
                                              (4096, 32, 200, 3)])
def test_page_tables(P, B, page, most, rows):
    rng = np.random.default_rng(B + page)
    print(f"tables: {B} requests, pages of {page}", flush=True)
    len_ = rng.integers(0, most + 1, B)
    add = rng.integers(0, rows + 1, B) * (rng.random(B) < 0.8)
    add[0] = rows                              # at least one row
    have = -(-len_ // page)
    need = -(-(len_ + add) // page)
    cols = need.max() + 2
    perm = rng.permutation(int(need.sum()) + 50)
    table = np.full((B, cols), -5, np.int32)
    at = 0
    for b in range(B):
        table[b, :have[b]] = perm[at:at + have[b]]
        at += have[b]
    free = perm[at:]
    got = same_tables(P, len_, add, page, free, table, int(add.sum()) + 13)
    assert got[5][2] == 0 and got[5][1] == (need - have).sum()
    same_tables(P, len_, add, page, free[:int((need - have).sum())], table, int(add.sum()))   # nothing to spare


@pytest.mark.parametrize("len_,add", [([0], [0]), ([0], [1]), ([31], [1]), ([32], [1]), ([32], [0]), ([33, 0, 0], [0, 0, 5]),
                                      ([5, 5, 5], [0, 0, 0]), ([-4, 7], [3, -2]), ([64, 64], [64, 65])])
def test_page_tables_edges(P, len_, add):
    table = np.full((len(len_), 6), 11, np.int32)
    same_tables(P, len_, add, 32, np.arange(20, 30), table, 140)


def test_page_tables_that_do_not_fit_change_nothing(P):
    len_, add = [30, 64, 1], [5, 1, 70]        # takes 1 + 1 + 2 pages, 76 rows
    table = np.arange(18, dtype=np.int32).reshape(3, 6)
    for free, cols, rows, flag in ((3, 6, 76, 1), (4, 6, 75, 2), (4, 2, 76, 4), (0, 2, 10, 7), (4, 6, 76, 0)):
        got = same_tables(P, len_, add, 32, np.arange(50, 50 + free), table[:, :cols].copy(), rows)
        assert got[5][2] == flag and got[5][3] == 4
        if flag:
            assert np.array_equal(got[0], table[:, :cols]) and np.all(got[4] == -1) and np.all(got[2] == 0)
    # sums that would pass 32 bits
    big = 2 ** 31 - 1
    for len_, add in (([5] * 40, [big] * 40), ([big] * 40, [0] * 40), ([big, big], [big, 7])):
        got = run_tables(P, len_, add, 32, np.arange(9), np.zeros((len(len_), 3), np.int32), 50)
        assert got[5][0] == 0 and got[5][2] & 4 and np.all(got[4] == -1) and np.array_equal(got[1], len_)


# --------------------------------------------------------------------------
# write and read
# --------------------------------------------------------------------------
def check_cache(dc, oc, slots):
    got = dc.read(slots)
    sc = dc.scales()
    for w in range(2):
        pages = np.unique(np.asarray(slots) // oc.page)
        assert np.array_equal(sc[w][pages], oc.scale[w][pages]), "scales"
        want = oc.values(w, slots)
        bad = got[w] != want
        assert not bad.any(), (f"{bad.sum()} of {bad.size} values of {'kv'[w]} differ, first at {np.argwhere(bad)[0]}: "
                               f"{got[w][bad][0]} for {want[bad][0]}")


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
@pytest.mark.parametrize("page,kv,hd", [(32, 1, 64), (32, 3, 128), (64, 2, 96), (128, 2, 32), (128, 1, 128),
                                        (64, 4, 64)])
def test_write_bit_for_bit(P, kind, page, kv, hd):
    """A prompt, single tokens and batches appended at random, growing scales,
    a page started anew, two requests in turn; every value after every call."""
    print(f"write: type {kind}, pages of {page}, {kv} x {hd}", flush=True)
    rng = np.random.default_rng(hd + page + kind)
    dc, oc = Q.DevCache(P, kind, page, 11, kv, hd), Q.Cache(kind, page, 11, kv, hd)
    tables = rng.permutation(11)[:10].reshape(2, 5)
    n = [0, 0]
    for step, m in enumerate([page + 7, 1, 1, 5, 1, 2 * page - 3, 1, 16, 1, 1, 9, 1]):
        b = step % 2
        m = min(m, 5 * page - n[b])
        pos = np.arange(n[b], n[b] + m)
        slot = tables[b][pos // page] * page + pos % page
        k, v = (rng.normal(0, 0.3 * (1 + step % 5), (m, kv * hd)).astype(np.float32) for _ in range(2))
        dc.write(k, v, slot, ldk=kv * hd + 4 * (step % 3), ldv=kv * hd + 8 * (step % 2))
        oc.write(k, v, slot)
        n[b] += m
        every = np.concatenate([tables[i][np.arange(n[i]) // page] * page + np.arange(n[i]) % page for i in range(2)])
        check_cache(dc, oc, every)
    # request 0 rolled back into the middle of a page and on, then to a page's start
    for keep in (page + 3, page):
        slot = tables[0][np.arange(keep, keep + 4) // page] * page + np.arange(keep, keep + 4) % page
        k, v = (rng.normal(0, 0.1, (4, kv * hd)).astype(np.float32) for _ in range(2))
        dc.write(k, v, slot)
        oc.write(k, v, slot)
        at = np.arange(keep + 4)
        check_cache(dc, oc, tables[0][at // page] * page + at % page)
    dc.free()


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
def test_write_special_values(P, kind):
    """Halves of a step exactly, one ulp either side of them, NaN, infinities,
    zeros, subnormals and pages below the smallest scale."""
    page, kv, hd = 32, 1, 32
    dc, oc = Q.DevCache(P, kind, page, 8, kv, hd), Q.Cache(kind, page, 8, kv, hd)
    rng = np.random.default_rng(kind)
    top = Q.TOP[kind]
    for p, scale in enumerate([1.0, np.float32(0.3), np.float32(1e-20), np.float32(7e20), np.float32(1 / 3.0)]):
        scale = np.float32(scale)
        codes = np.arange(-126.5, 127.0, 1.0) if kind == Q.INT8 else np.concatenate(
            [s * (Q.E4M3_VALUES[:126] + Q.E4M3_VALUES[1:127]) / 2 for s in (1, -1)])
        x = (rng.choice(codes, (page, hd)) * scale).astype(np.float32)
        x[::3] = np.nextafter(x[::3], np.float32(np.inf))
        x[1::3] = np.nextafter(x[1::3], np.float32(-np.inf))
        x[0, 0] = np.float32(top) * scale
        v = x.copy()
        v[3, 5], v[4, 6], v[5, 7], v[6, :] = np.nan, np.inf, -np.inf, 0
        slot = p * page + np.arange(page)
        dc.write(x, v, slot)
        oc.write(x, v, slot)
        check_cache(dc, oc, slot)
    # zeros; values too small for a scale; a page of NaN alone; then growth from a scale of zero
    for p, x in ((5, np.zeros((4, hd))), (6, np.full((4, hd), 2.0 ** -101)), (7, np.full((4, hd), np.nan))):
        slot = p * page + np.arange(4)
        x = x.astype(np.float32)
        dc.write(x, x, slot)
        oc.write(x, x, slot)
        check_cache(dc, oc, slot)
        y = rng.normal(0, 1, (3, hd)).astype(np.float32)
        dc.write(y, y, p * page + 4 + np.arange(3))
        oc.write(y, y, p * page + 4 + np.arange(3))
        check_cache(dc, oc, p * page + np.arange(7))
    dc.free()


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
def test_write_any_order_and_foreign_slots(P, kind):
    """Rows in any order, slots of no page, the same slot twice, one request's
    rows among another's; pages that no row names keep every byte."""
    page, kv, hd, pool = 64, 2, 64, 9
    dc, oc = Q.DevCache(P, kind, page, pool, kv, hd), Q.Cache(kind, page, pool, kv, hd)
    rng = np.random.default_rng(11)
    first = np.arange(6 * page)                     # pages 0..5 full, 6..8 untouched
    for lo in range(0, len(first), 100):
        s = first[lo:lo + 100]
        k, v = (rng.normal(0, 1, (len(s), kv * hd)).astype(np.float32) for _ in range(2))
        dc.write(k, v, s)
        oc.write(k, v, s)
    before = dc.bytes()
    slot = np.concatenate([rng.permutation(np.arange(70, 100)), [-1, pool * page, pool * page + 5, 2 ** 31 - 1, -2 ** 31],
                           [200, 200, 210, 200], [130, 71, 131, 75], [-1]])
    k, v = (rng.normal(0, 2, (len(slot), kv * hd)).astype(np.float32) for _ in range(2))
    dc.write(k, v, slot)
    oc.write(k, v, slot)
    check_cache(dc, oc, np.arange(6 * page))
    after = dc.bytes()
    for w in range(2):
        for p in (0, 4, 5, 6, 7, 8):
            assert np.array_equal(before[w][p], after[w][p]), f"page {p} changed"
    # rows of no slot are left as they were by the read
    got = dc.read(np.array([-1, 70, pool * page, 2 ** 31 - 1]), fill=42.0)
    assert np.all(got[0][[0, 2, 3]] == 42.0) and np.all(got[1][[0, 2, 3]] == 42.0)
    assert np.array_equal(got[0][1:2], oc.values(0, [70]))
    dc.free()


def test_write_many_rows(P):
    """The most rows of one call: a batch of single tokens, and a long prompt."""
    page, kv, hd = 32, 1, 64
    rng = np.random.default_rng(3)
    print("write: 8192 rows", flush=True)
    dc, oc = Q.DevCache(P, Q.INT8, page, 8192, kv, hd), Q.Cache(Q.INT8, page, 8192, kv, hd)
    k, v = (rng.normal(0, 1, (8192, hd)).astype(np.float32) for _ in range(2))
    own_page = rng.permutation(8192) * page
    dc.write(k, v, own_page)
    oc.write(k, v, own_page)
    check_cache(dc, oc, own_page)
    prompt = 5 + np.arange(8192)
    dc.write(k, v, prompt)
    oc.write(k, v, prompt)
    check_cache(dc, oc, prompt)
    dc.free()


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------
def filled(P, kind, page, pool, kv, hd, rng, garbage=True):
    """A cache of random codes and scales on both sides."""
    dc, oc = Q.DevCache(P, kind, page, pool, kv, hd), Q.Cache(kind, page, pool, kv, hd)
    for w in range(2):
        raw = rng.integers(0, 256, (pool, kv, page, hd), dtype=np.uint8)
        if kind == Q.E4M3:
            raw[(raw & 127) == 127] = 3
            val = Q.E4M3_VALUES[raw] 
        else:
            raw[raw == 0] = 5
            val = raw.astype(np.float64) - 128
        oc.code[w] = val
        oc.scale[w] = (rng.uniform(0.5, 2, (pool, kv)) * (0.012 if kind == Q.INT8 else 0.004)).astype(np.float32)
        t, d = np.arange(page)[:, None], np.arange(hd)[None, :]
        if w == 0:
            at = t // 32 * 32 * hd + d // 32 * 1024 + (d // 8 % 4 * 16 + t % 16) * 16 + t // 16 % 2 * 8 + d % 8
        else:
            at = t // 32 * 32 * hd + d // 32 * 1024 + (t // 4 % 4 * 16 + d % 16) * 16 + d // 16 % 2 * 8 + \
                t // 16 % 2 * 4 + t % 4
        phys = np.zeros((pool, kv, page * hd), np.uint8)
        phys[:, :, at.reshape(-1)] = raw.reshape(pool, kv, -1)
        base = (dc.s.k, dc.s.v)[w]
        assert P.vxh_upload(C.c_void_p(base), N._ptr(phys), phys.nbytes, None) == 0
        sc = oc.scale[w]
        assert P.vxh_upload(C.c_void_p((dc.s.ks, dc.s.vs)[w]), N._ptr(sc), sc.nbytes, None) == 0
    return dc, oc


def check_attend(P, dc, oc, q, row0, len_, table, H, cap, **kw):
    got = Q.run_attend(P, dc, q, row0, len_, table, H, cap, **kw)
    fill = kw.get("fill", -3.0)
    want, tol = Q.attend(q, oc, row0, len_, table, H, cap, np.full(got.shape, fill))
    d = np.abs(got - want)
    assert np.all(np.isfinite(got)), "not finite"
    assert np.all(d.max(axis=1) <= tol), f"row {np.argmax(d.max(axis=1) - tol)}: {d.max()} past {tol[np.argmax(d.max(axis=1) - tol)]}"
    return got


def ragged(rng, lens, adds, page, extra_cols=0):
    need = [-(-n // page) for n in lens]
    pool = sum(need) + 3
    perm = rng.permutation(pool)
    table = np.full((len(lens), max(max(need), 1) + extra_cols), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return pool, table, np.concatenate([[0], np.cumsum(adds)]).astype(np.int32)


BATCHES = [
    # lengths, rows, query heads, kv heads, head size, page, cap
    ([1], [1], 1, 1, 32, 32, 0),
    ([2048], [1], 32, 4, 64, 32, 0),
    ([2057], [9], 28, 4, 128, 64, 0),
    ([1, 2, 31, 32, 33, 63, 64, 65, 100], [1] * 9, 4, 2, 128, 32, 0),
    ([16, 17, 5, 300], [16, 17, 5, 16], 3, 1, 96, 32, 0),
    ([0, 40, 0, 7], [0, 3, 0, 7], 8, 8, 64, 64, 0),
    ([129, 1000, 3], [4, 2, 3], 7, 7, 32, 128, 0),
    ([700, 90], [1, 5], 8, 2, 128, 64, 100),
    ([200], [200], 4, 2, 64, 32, 0),
    ([333, 400], [333, 150], 4, 4, 128, 64, 0),
    ([500, 70, 260, 1], [300, 1, 130, 1], 14, 2, 64, 32, 0),
    ([260, 515], [129, 257], 3, 3, 96, 128, 200),
    ([140], [140], 16, 1, 32, 32, 64),
    ([3000, 5, 17, 1200], [1, 1, 2, 1], 4, 4, 128, 32, 2049),
    ([40] * 70, [2] * 70, 4, 2, 64, 32, 0),
    # enough query tiles for the prompt kernel: of four streams, of two
    ([130], [130], 64, 64, 32, 32, 0),
    ([1100], [97], 224, 32, 32, 64, 0),
    ([333], [129], 64, 64, 96, 128, 200),
    ([2049, 40, 66, 300], [64, 0, 66, 1], 64, 64, 64, 32, 2049),
    ([70, 400, 5, 31], [65, 300, 1, 31], 64, 64, 64, 64, 0),
    ([300, 700], [200, 200], 128, 16, 32, 128, 0),
    ([500], [390], 64, 64, 128, 64, 77),
    ([90] * 40, [70] * 40, 16, 8, 32, 32, 0),
]


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
@pytest.mark.parametrize("case", range(len(BATCHES)))
def test_attention(P, kind, case):
    lens, adds, H, KV, hd, page, cap = BATCHES[case]
    print(f"attention: type {kind}, lengths {lens[:9]}, rows {adds[:9]}, {H}/{KV} heads of {hd}, page {page}, cap {cap}",
          flush=True)
    rng = np.random.default_rng(case + 100 * kind)
    pool, table, row0 = ragged(rng, lens, adds, page, extra_cols=case % 3)
    dc, oc = filled(P, kind, page, pool, KV, hd, rng)
    q = rng.normal(0, 1.5, (row0[-1], H * hd)).astype(np.float32)
    got = check_attend(P, dc, oc, q, row0, lens, table, H, cap, max_rows=row0[-1] + 5, ld_extra=4 * (case % 3),
                       out_extra=8 * (case % 2))
    # the hint changes which kernel runs, not what comes out of a row beyond rounding
    for hint in (1, 100000):
        check_attend(P, dc, oc, q, row0, lens, table, H, cap, max_seq_rows=hint)
    # the same call gives the same bits
    again = Q.run_attend(P, dc, q, row0, lens, table, H, cap, max_rows=row0[-1] + 5)
    assert np.array_equal(got, again)
    dc.free()


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
@pytest.mark.parametrize("rows,H,KV", [(1, 6, 2), (9, 6, 2), (150, 6, 2), (150, 64, 64)])
def test_attention_ignores_what_no_row_reads(P, kind, rows, H, KV):
    """Bytes of every kind (e4m3 NaN among them) behind the last token, NaN
    scales on pages behind it, garbage in the table's unused columns."""
    page, hd, n = 64, 64, 203
    rng = np.random.default_rng(rows)
    pool, table, row0 = ragged(rng, [n], [rows], page, extra_cols=2)
    dc, oc = filled(P, kind, page, pool, KV, hd, rng)
    q = rng.normal(0, 1, (rows, H * hd)).astype(np.float32)
    want = check_attend(P, dc, oc, q, row0, [n], table, H, 0)
    table[0, -2:] = [2 ** 31 - 1, -77]
    raw = dc.bytes()
    last = table[0, n // page]
    t, d = np.arange(page)[:, None], np.arange(hd)[None, :]
    at = [t // 32 * 32 * hd + d // 32 * 1024 + (d // 8 % 4 * 16 + t % 16) * 16 + t // 16 % 2 * 8 + d % 8,
          t // 32 * 32 * hd + d // 32 * 1024 + (t // 4 % 4 * 16 + d % 16) * 16 + d // 16 % 2 * 8 + t // 16 % 2 * 4 + t % 4]
    for byte in (0x7F, 0xFF, 0x80):
        for w in range(2):
            for h in range(KV):
                page_bytes = raw[w][last, h].copy()
                page_bytes[at[w][n % page:].reshape(-1)] = byte
                dc.put(w, last, h, page_bytes)
            for p in range(pool):
                if p not in table[0, :-(-n // page)]:
                    dc.put_scale(w, p, 0, np.nan)
        assert np.array_equal(Q.run_attend(P, dc, q, row0, [n], table, H, 0), want), hex(byte)
    # and the positions a cap cuts off
    capped = check_attend(P, dc, oc, q, row0, [n], table, H, 65)
    for h in range(KV):
        for w in range(2):
            dc.put(w, table[0, 2], h, np.full(page * hd, 0x7F, np.uint8))
            dc.put_scale(w, table[0, 2], h, np.inf)
    assert np.array_equal(Q.run_attend(P, dc, q, row0, [n], table, H, 65), capped)
    dc.free()


@pytest.mark.parametrize("rows,H,KV", [(1, 4, 2), (5, 4, 2), (140, 4, 2), (70, 48, 48)])
def test_attention_of_lengths_and_tables_that_lie(P, rows, H, KV):
    """Table entries that are no page, lengths past the table, fewer tokens
    than rows, negative lengths: rows read what there is, or are zeros."""
    page, hd = 32, 64
    rng = np.random.default_rng(rows + 1)
    dc, oc = filled(P, Q.INT8, page, 12, KV, hd, rng)
    table = np.array([[3, -1, 5, 7, 9], [1, 2, 12, 2 ** 31 - 1, 4], [0, 6, 8, 10, 11], [-1, -1, -1, -1, -1]], np.int32)
    row0 = np.array([0, rows, 2 * rows, 3 * rows, 4 * rows], np.int32)
    q = rng.normal(0, 1, (4 * rows, H * hd)).astype(np.float32)
    for len_ in ([150, 160, 400, 100], [140, 2 ** 31 - 1, 3, -5], [0, 1, 2 ** 30, 64]):
        got = Q.run_attend(P, dc, q, row0, len_, table, H, 0)
        want, tol = Q.attend(q, oc, row0, len_, table, H, 0, np.full(got.shape, -3.0))
        assert np.all(np.abs(got - want).max(axis=1) <= tol)
    assert np.all(got[:rows - 1] == 0)          # length 0: only zeros
    # row starts out of order or past the rows: no access out of bounds, the call ends
    for bad in ([0, 3, 1, 4 * rows, 2], [-5, 1, 10 ** 6, 2 ** 31 - 1, -1], [4 * rows] * 5):
        Q.run_attend(P, dc, q, np.array(bad, np.int32), [100] * 4, table, H, 0, max_seq_rows=rows)
    dc.free()


@pytest.mark.parametrize("rows,H,KV", [(3, 2, 1), (66, 96, 96)])
def test_attention_scores_far_apart(P, rows, H, KV):
    """Scores over a range that underflows every probability but one, large
    and tiny queries, scales that differ by 2^40 between pages."""
    page, hd, n = 32, 64, 1000 if rows == 3 else 300
    rng = np.random.default_rng(8)
    pool, table, row0 = ragged(rng, [n], [rows], page)
    for kind in (Q.INT8, Q.E4M3):
        dc, oc = filled(P, kind, page, pool, KV, hd, rng)
        # (at 1e9 a score's own fp32 rounding is past every other score: 64 bits
        # say which token wins, and no tolerance but the largest value's bounds it)
        for qs in (1e9, 1e25, 1e-30, 40.0, 3000.0):
            q = (rng.normal(0, 1, (rows, H * hd)) * qs).astype(np.float32)
            check_attend(P, dc, oc, q, row0, [n], table, H, 0)
        q[1] = 0
        check_attend(P, dc, oc, q, row0, [n], table, H, 0)
        sc = (2.0 ** rng.integers(-30, 10, (pool, KV))).astype(np.float32)
        oc.scale[1] = sc
        assert P.vxh_upload(C.c_void_p(dc.s.vs), N._ptr(sc), sc.nbytes, None) == 0
        check_attend(P, dc, oc, rng.normal(0, 1, (rows, H * hd)).astype(np.float32), row0, [n], table, H, 0)
        dc.free()


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
def test_cache_past_4_gib(P, kind):
    """The first and the last pages of a pool whose keys alone pass 32 bits."""
    page, kv, hd = 128, 8, 128
    pool = (1 << 32) // (page * kv * hd) + 200
    print(f"pool of {pool} pages, {pool * page * kv * hd / 2**30:.2f} GiB of keys", flush=True)
    dc = Q.DevCache(P, kind, page, pool, kv, hd)
    rng = np.random.default_rng(1)
    small = Q.Cache(kind, page, 4, kv, hd)
    pages = np.array([0, pool - 1, (1 << 32) // (page * kv * hd), pool - 2])
    k, v = (rng.normal(0, 1, (4 * page, kv * hd)).astype(np.float32) for _ in range(2))
    slot = np.arange(4 * page)
    big = (pages[slot // page] * page + slot % page).astype(np.int32)
    dc.write(k, v, big)
    small.write(k, v, slot)
    got = dc.read(big)
    for w in range(2):
        assert np.array_equal(got[w], small.values(w, slot))
    q = rng.normal(0, 1, (133, 8 * hd)).astype(np.float32)
    row0, len_ = np.array([0, 1, 4, 133]), [500, 200, 512]
    table = np.stack([pages[[0, 1, 2, 3]], pages[[1, 3, 0, 2]], pages[[2, 0, 3, 1]]]).astype(np.int32)
    idx = {p: i for i, p in enumerate(pages)}
    out = Q.run_attend(P, dc, q, row0, len_, table, 8, 0)
    want, tol = Q.attend(q, small, row0, len_, np.vectorize(idx.get)(table), 8, 0, np.zeros(out.shape))
    assert np.all(np.abs(out - want).max(axis=1) <= tol)
    dc.free()


def test_long_context(P):
    """A hundred thousand tokens, one row and a few, over many segments."""
    page, KV, H, hd, n = 128, 1, 2, 64, 100003
    rng = np.random.default_rng(2)
    pool, table, row0 = ragged(rng, [n, 70], [2, 1], page)
    dc, oc = filled(P, Q.INT8, page, pool, KV, hd, rng)
    q = rng.normal(0, 1, (3, H * hd)).astype(np.float32)
    check_attend(P, dc, oc, q, row0, [n, 70], table, H, 0)
    dc.free()


# --------------------------------------------------------------------------
# steps of serving
# --------------------------------------------------------------------------
class Server:
    """A pool, a table and the arrays of a step, sized once, with the step's
    three calls on one stream; the lengths live on the device between steps."""

    def __init__(self, P, kind, page, pool, cols, B, H, KV, hd, max_rows, stream):
        self.P, self.B, self.H, self.KV, self.hd, self.R = P, B, H, KV, hd, max_rows
        self.page, self.pool, self.cols, self.stream = page, pool, cols, stream
        self.dc, self.oc = Q.DevCache(P, kind, page, pool, KV, hd), Q.Cache(kind, page, pool, KV, hd)
        w, kw = H * hd, KV * hd
        shape = dict(len=B, add=B, free=pool, table=B * cols, len_out=B, row0=B + 1, pos=max_rows, slot=max_rows,
                     counts=4, q=max_rows * w, k=max_rows * kw, v=max_rows * kw, out=max_rows * w)
        self.d = {n: N.DevBuf(P, np.zeros(c, np.int32)) for n, c in shape.items()}
        self.ws = Q.Workspace()
        n = P.vxh_attention_kvq_workspace_floats(max_rows, B, H, KV, hd)
        assert P.vxh_workspace_alloc(C.byref(self.ws), 32, n) == 0
        self.len = np.zeros(B, np.int32)
        self.free = np.random.default_rng(pool).permutation(pool).astype(np.int32)
        self.table = np.full((B, cols), -1, np.int32)
        self.put("table", self.table)

    def put(self, name, a):
        a = np.ascontiguousarray(a)
        assert a.nbytes <= self.d[name].nbytes
        assert self.P.vxh_upload(self.d[name].ptr, N._ptr(a), a.nbytes, self.stream) == 0

    def launch(self):
        P, d = self.P, self.d
        w, kw = self.H * self.hd, self.KV * self.hd
        assert P.vxh_page_tables(d["len"].ptr, d["add"].ptr, self.B, self.page, d["free"].ptr, self.n_free,
                                 d["table"].ptr, self.cols, d["len_out"].ptr, d["row0"].ptr, d["pos"].ptr, d["slot"].ptr,
                                 self.R, d["counts"].ptr, self.stream) == 0, P.vxh_last_error()
        assert P.vxh_kvq_write(self.dc.ref, d["k"].ptr, kw, d["v"].ptr, kw, d["slot"].ptr, self.R, self.stream) == 0
        assert P.vxh_attention_kvq(d["q"].ptr, w, d["row0"].ptr, d["len_out"].ptr, self.B, self.R, self.hint,
                                   d["table"].ptr, self.cols, self.H, self.dc.ref, 0, d["out"].ptr, w, C.byref(self.ws),
                                   self.stream) == 0, P.vxh_last_error()

    def inputs(self, rng, add):
        self.add = np.asarray(add, np.int32)
        self.q = rng.normal(0, 1, (self.R, self.H * self.hd)).astype(np.float32)
        self.k, self.v = (rng.normal(0, rng.uniform(0.5, 2), (self.R, self.KV * self.hd)).astype(np.float32)
                          for _ in range(2))
        pad = np.full(self.pool, -1, np.int32)
        pad[:len(self.free)] = self.free
        for n, a in (("len", self.len), ("add", self.add), ("free", pad), ("q", self.q), ("k", self.k), ("v", self.v),
                     ("out", np.full((self.R, self.H * self.hd), -3.0, np.float32))):
            self.put(n, a)

    def check(self, what):
        P = self.P
        assert P.vxh_stream_sync(self.stream) == 0
        table, len_, row0, pos, slot, counts = Q.tables(self.len, self.add, self.page, self.free, self.table, self.R)
        for n, want in (("table", table), ("len_out", len_), ("row0", row0), ("slot", slot), ("counts", counts)):
            assert np.array_equal(self.d[n].get(np.int32, want.size), want.reshape(-1)), (what, n)
        self.oc.write(self.k, self.v, slot)
        got = self.d["out"].get(np.float32, self.q.size).reshape(self.q.shape)
        want, tol = Q.attend(self.q, self.oc, row0, len_, table, self.H, 0, np.full(got.shape, -3.0))
        d = np.abs(got - want).max(axis=1)
        assert np.all(d <= tol), (what, int(np.argmax(d - tol)), d.max())
        live = slot[slot >= 0]
        if len(live):
            check_cache(self.dc, self.oc, live)
        self.table, self.len, self.free = table, len_, self.free[counts[1]:]

    def release(self, b, keep):
        """Request b rolled back to keep tokens; its further pages return."""
        have = -(-int(self.len[b]) // self.page)
        kept = -(-keep // self.page)
        self.free = np.concatenate([self.free, self.table[b, kept:have]])
        self.len[b] = keep

    def close(self):
        for b in self.d.values():
            b.free()
        self.P.vxh_workspace_free(C.byref(self.ws))
        self.dc.free()


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
@pytest.mark.parametrize("graph", [False, True])
def test_serving_steps(P, kind, graph):
    """Prompts, decoding, verify batches with roll-back, a step that does not
    fit, a request that leaves: each step's tables, cache and attention
    against the oracle; the same steps from one captured graph."""
    s = C.c_void_p()
    assert P.vxh_stream_create(C.byref(s)) == 0
    sv = Server(P, kind, 32, 40, 12, 5, 6, 2, 64, 220, s)
    rng = np.random.default_rng(17)
    sv.n_free = sv.pool if graph else None
    sv.hint = 200
    g = C.c_void_p()
    if graph:
        # every replay offers the whole array; entries behind the free pages are -1,
        # so a step that needs more of them than there are must not be made
        sv.inputs(rng, [1] * 5)
        assert P.vxh_capture_begin(s) == 0
        sv.launch()
        assert P.vxh_capture_end(s, C.byref(g)) == 0, P.vxh_last_error()
    steps = [[70, 3, 0, 1, 33], [1, 1, 1, 1, 1], [9, 0, 150, 1, 1], [1, 1, 1, 1, 1], [1, 9, 1, 9, 1], [0, 0, 0, 0, 0],
             [1, 2, 3, 4, 5], [1, 1, 1, 30, 1]]
    for i, add in enumerate(steps):
        print(f"step {i}: rows {add}", flush=True)
        if i == 3:
            sv.release(0, int(sv.len[0]) - 6)       # six drafts refused
        if i == 6:
            sv.release(2, 0)                        # a conversation ends
        sv.inputs(rng, add)
        if graph:
            assert P.vxh_graph_launch(g, s) == 0
        else:
            sv.n_free = len(sv.free)
            sv.launch()
        sv.check(f"step {i}")
    if not graph:
        sv.n_free = 1
        sv.inputs(rng, [100, 1, 1, 1, 1])           # does not fit: nothing happens
        before = sv.dc.bytes()
        sv.launch()
        assert P.vxh_stream_sync(s) == 0
        assert sv.d["counts"].get(np.int32, 4)[2] == 1
        assert np.all(sv.d["out"].get(np.float32, sv.q.size) == -3.0)
        assert all(np.array_equal(a, b) for a, b in zip(before, sv.dc.bytes()))
    else:
        assert P.vxh_graph_destroy(g) == 0
    sv.close()
    assert P.vxh_stream_destroy(s) == 0
