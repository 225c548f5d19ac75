"""The paged 8-bit KV cache's calls as a server makes them: batches of hundreds
and thousands of requests, calls on two streams at once, a workspace shared in
turn with another attention, replayed graphs that need both attention kernels,
shared pages, padded batches and rows that are not numbers (tolerance derived
in _kvq.attend)."""
import ctypes as C

import numpy as np
import pytest

import _kvq as Q
import _native as N
from test_gpu_kvq import Server, check_attend, filled, ragged

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def P():
    if not N.product_available():
        pytest.fail("product library not built")
    L = Q.bind(N.bind_vxh(N.product()))
    assert L.vxh_init() == 0, L.vxh_last_error()
    return L


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
@pytest.mark.parametrize("B,most,H,KV,long_rows", [(257, 200, 4, 2, 1), (600, 40, 8, 8, 20), (4096, 70, 2, 1, 3),
                                                   (700, 90, 64, 16, 90)])
def test_many_requests(P, kind, B, most, H, KV, long_rows):
    """Runs of requests per thread, some without rows, one much longer than the rest."""
    page, hd = 32, 32
    print(f"attention: type {kind}, {B} requests, {H}/{KV} heads", flush=True)
    rng = np.random.default_rng(B + kind)
    lens = rng.integers(1, most + 1, B)
    lens[B // 3] = 1500
    adds = np.where(rng.random(B) < 0.3, 0, 1)
    adds[rng.integers(0, B, 4)] = long_rows
    adds = np.minimum(adds, lens)
    adds[-5:] = 0                                       # the last requests stand still
    pool, table, row0 = ragged(rng, lens, adds, page)
    dc, oc = filled(P, kind, page, pool, KV, hd, rng)
    q = rng.normal(0, 1.5, (row0[-1], H * hd)).astype(np.float32)
    a = check_attend(P, dc, oc, q, row0, lens, table, H, 0, max_rows=row0[-1] + 3)
    assert np.array_equal(a, Q.run_attend(P, dc, q, row0, lens, table, H, 0, max_rows=row0[-1] + 3))
    check_attend(P, dc, oc, q, row0, lens, table, H, 0, max_seq_rows=1)
    dc.free()


class Call:
    """An attention call's buffers, kept, on a stream of its own."""

    def __init__(self, P, dc, q, row0, len_, table, H, ws=None):
        self.P, self.dc, self.H, self.q, self.n, self.cols = P, dc, H, q, len(len_), table.shape[1]
        self.m = int(np.diff(row0).max())
        self.s = C.c_void_p()
        assert P.vxh_stream_create(C.byref(self.s)) == 0
        self.bufs = [N.DevBuf(P, np.ascontiguousarray(a)) for a in (
            q, np.asarray(row0, np.int32), np.asarray(len_, np.int32), table.astype(np.int32), np.full_like(q, -3.0))]
        self.own = ws is None
        self.ws = ws or Q.Workspace()
        if self.own:
            n = P.vxh_attention_kvq_workspace_floats(len(q), self.n, H, dc.kv, dc.hd)
            assert P.vxh_workspace_alloc(C.byref(self.ws), 32, n) == 0

    def launch(self, stream=None):
        b, w = self.bufs, self.q.shape[1]
        assert self.P.vxh_attention_kvq(b[0].ptr, w, b[1].ptr, b[2].ptr, self.n, len(self.q), self.m, b[3].ptr, self.cols,
                                        self.H, self.dc.ref, 0, b[4].ptr, w, C.byref(self.ws), stream or self.s) == 0

    def result(self, stream=None):
        assert self.P.vxh_stream_sync(stream or self.s) == 0
        return self.bufs[4].get(np.float32, self.q.size).reshape(self.q.shape)

    def counters(self):
        c = np.ones(1024, np.int32)
        assert self.P.vxh_download(N._ptr(c), C.c_void_p(self.ws.acc + 8 * self.ws.acc_elems), c.nbytes, None) == 0
        return c

    def close(self):
        for b in self.bufs:
            b.free()
        if self.own:
            self.P.vxh_workspace_free(C.byref(self.ws))
        assert self.P.vxh_stream_destroy(self.s) == 0


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
def test_two_streams_at_once(P, kind):
    """Calls on two streams over one cache, each with its workspace, give what
    each gives alone, and every counter is back at zero."""
    page, hd, H, KV = 64, 128, 8, 2
    rng = np.random.default_rng(4)
    pool, table, _ = ragged(rng, [9000, 700, 64, 3000], [1] * 4, page)
    dc, oc = filled(P, kind, page, pool, KV, hd, rng)
    calls = []
    for adds, order in (([3, 1, 1, 9], [0, 1, 2, 3]), ([40, 64, 1, 2], [3, 1, 2, 0])):
        row0 = np.concatenate([[0], np.cumsum(adds)])
        len_ = np.array([9000, 700, 64, 3000])[order]
        q = rng.normal(0, 1, (row0[-1], H * hd)).astype(np.float32)
        calls.append(Call(P, dc, q, row0, len_, table[order], H))
        check_attend(P, dc, oc, q, row0, len_, table[order], H, 0)
    alone = []
    for c in calls:
        c.launch()
        alone.append(c.result())
    for _ in range(20):
        for c in calls:
            c.launch()
    for c, want in zip(calls, alone):
        assert np.array_equal(c.result(), want)
        assert not c.counters().any()
        c.close()
    dc.free()


def test_workspace_in_turn_with_another_attention(P):
    """One workspace serves both attentions on one stream, each call after the other."""
    page, hd, H, KV, n = 32, 64, 4, 2, 5000
    rng = np.random.default_rng(9)
    pool, table, row0 = ragged(rng, [n], [2], page)
    dc, oc = filled(P, Q.INT8, page, pool, KV, hd, rng)
    q = rng.normal(0, 1, (2, H * hd)).astype(np.float32)
    want = check_attend(P, dc, oc, q, row0, [n], table, H, 0)
    ws = Q.Workspace()
    P.vxh_attention_workspace_floats.restype = C.c_size_t
    floats = max(P.vxh_attention_workspace_floats(2, n, 0, H, KV, hd),
                 P.vxh_attention_kvq_workspace_floats(2, 1, H, KV, hd))
    assert P.vxh_workspace_alloc(C.byref(ws), 32, floats) == 0
    c = Call(P, dc, q, row0, [n], table, H, ws=ws)
    kv = [N.DevBuf(P, rng.normal(0, 1, (n, KV * hd)).astype(np.float32)) for _ in range(2)]
    other = N.DevBuf(P, np.zeros((2, H * hd), np.float32))
    seen = []
    for _ in range(4):
        c.launch()
        assert P.vxh_attention(c.bufs[0].ptr, 2, n - 2, n, H, KV, hd, 0, kv[0].ptr, kv[1].ptr, other.ptr, H * hd,
                               C.byref(ws), c.s) == 0, P.vxh_last_error()
        c.launch()
        assert np.array_equal(c.result(), want)
        seen.append(other.get(np.float32, q.size))
        assert np.array_equal(seen[0], seen[-1]) and np.abs(seen[0]).max() > 0
    c.close()
    for b in kv + [other]:
        b.free()
    P.vxh_workspace_free(C.byref(ws))
    dc.free()


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
def test_graph_of_both_attention_kernels(P, kind):
    """One captured step whose replays hold prompts, single tokens, both, and
    nothing; eager work and synchronizations stand between them."""
    s = C.c_void_p()
    assert P.vxh_stream_create(C.byref(s)) == 0
    sv = Server(P, kind, 32, 48, 14, 4, 64, 64, 32, 220, s)
    rng = np.random.default_rng(23)
    sv.n_free, sv.hint = sv.pool, 200                   # 64 heads x 220 rows: tiles enough for the prompt kernel
    g = C.c_void_p()
    sv.inputs(rng, [1] * 4)
    assert P.vxh_capture_begin(s) == 0
    sv.launch()
    assert P.vxh_capture_end(s, C.byref(g)) == 0, P.vxh_last_error()
    for i, add in enumerate([[200, 3, 0, 1], [1, 1, 1, 1], [0, 0, 0, 0], [1, 100, 64, 1], [2, 1, 65, 70], [1, 1, 1, 1]]):
        print(f"replay {i}: rows {add}", flush=True)
        sv.inputs(rng, add)
        assert P.vxh_graph_launch(g, s) == 0
        sv.check(f"replay {i}")
    assert P.vxh_graph_destroy(g) == 0
    sv.close()
    assert P.vxh_stream_destroy(s) == 0


@pytest.mark.parametrize("rows,H,KV", [(1, 4, 2), (7, 6, 2), (130, 64, 64)])
def test_row_starts_and_padding(P, rows, H, KV):
    """Rows that begin behind others, far fewer of them than max_rows: those
    in front and behind stay as they were."""
    page, hd, n = 32, 32, 300
    rng = np.random.default_rng(rows)
    pool, table, _ = ragged(rng, [n], [rows], page)
    dc, oc = filled(P, Q.E4M3, page, pool, KV, hd, rng)
    q = rng.normal(0, 1, (rows + 8, H * hd)).astype(np.float32)
    for B in (1, 2):                                    # (a second request without rows)
        row0 = np.array([3] + [3 + rows] * B, np.int32)
        lens, tab = [n] * B, np.repeat(table, B, axis=0)
        got = check_attend(P, dc, oc, q, row0, lens, tab, H, 0, max_rows=rows + 400)
        assert np.all(got[:3] == -3.0) and np.all(got[3 + rows:] == -3.0)
    dc.free()


def test_pages_shared_by_requests(P):
    """A common prompt's pages in every request's table, and one page twice in a row of it."""
    page, hd, H, KV = 32, 64, 8, 2
    rng = np.random.default_rng(31)
    dc, oc = filled(P, Q.INT8, page, 20, KV, hd, rng)
    table = np.array([[4, 5, 6, b + 7, 6, 4] for b in range(6)], np.int32)
    lens = [97, 128, 150, 192, 96, 33]
    adds = [1, 9, 70, 1, 30, 2]
    row0 = np.concatenate([[0], np.cumsum(adds)]).astype(np.int32)
    q = rng.normal(0, 1, (row0[-1], H * hd)).astype(np.float32)
    check_attend(P, dc, oc, q, row0, lens, table, H, 0)
    dc.free()


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
@pytest.mark.parametrize("rows,H,KV", [(3, 6, 2), (70, 64, 64)])
def test_rows_that_are_not_numbers_stand_alone(P, kind, rows, H, KV):
    """A query with NaN or infinities changes no other row or head."""
    page, hd, n = 64, 64, 260
    rng = np.random.default_rng(5)
    pool, table, row0 = ragged(rng, [n], [rows], page)
    dc, oc = filled(P, kind, page, pool, KV, hd, rng)
    q = rng.normal(0, 1, (rows, H * hd)).astype(np.float32)
    want, tol = Q.attend(q, oc, row0, [n], table, H, 0, np.zeros(q.shape))
    q[1, 2 * hd + 5], q[1, 3 * hd], q[2, 7] = np.nan, np.inf, -np.inf
    got = Q.run_attend(P, dc, q, row0, [n], table, H, 0)
    ok = np.ones(q.shape, bool)
    ok[1, 2 * hd:4 * hd], ok[2, :hd] = False, False
    assert np.all((np.abs(got - want) <= tol[:, None])[ok])
    dc.free()


@pytest.mark.parametrize("rows,H,KV", [(2, 2, 1), (66, 96, 96)])
@pytest.mark.parametrize("size", [1e36, 1e-28])
def test_values_at_the_ends_of_fp32(P, rows, H, KV, size):
    """Values near fp32's largest, and pages whose scale is near the smallest
    that a write makes (2^-100 / 448): the sums neither overflow nor vanish."""
    page, hd, n = 32, 64, 300
    rng = np.random.default_rng(12)
    pool, table, row0 = ragged(rng, [n], [rows], page)
    for kind in (Q.INT8, Q.E4M3):
        dc, oc = filled(P, kind, page, pool, KV, hd, rng)
        sc = (rng.uniform(0.5, 1, (pool, KV)) * size / Q.TOP[kind]).astype(np.float32)
        oc.scale[1] = sc
        assert P.vxh_upload(C.c_void_p(dc.s.vs), N._ptr(sc), sc.nbytes, None) == 0
        q = (rng.normal(0, 1, (rows, H * hd))).astype(np.float32)
        check_attend(P, dc, oc, q, row0, [n], table, H, 0)
        check_attend(P, dc, oc, q, row0, [n], table, H, 0, max_seq_rows=1)
        dc.free()


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
def test_most_rows_of_a_call(P, kind):
    """The largest max_rows with a few rows in it, and with all but a few of them
    one prompt's."""
    page, hd, R = 32, 32, 1 << 18
    rng = np.random.default_rng(77)
    for adds in ([2, 1, 70], [1, R - 9, 3]):
        lens = [300, max(adds[1], 40), 90]
        print(f"attention: type {kind}, rows {adds} of {R}", flush=True)
        pool, table, row0 = ragged(rng, lens, adds, page)
        dc, oc = filled(P, kind, page, pool, 1, hd, rng)
        q = rng.normal(0, 1, (row0[-1], hd)).astype(np.float32)
        got = Q.run_attend(P, dc, q, row0, lens, table, 1, 100, max_rows=R, max_seq_rows=R)
        assert np.all(got[row0[-1]:] == -3.0)
        # 64 bits for the requests at both ends and for rows here and there between
        pick = [0, 2] if adds[1] > 1000 else [0, 1, 2]
        for b in pick:
            rows = slice(row0[b], row0[b + 1])
            want, tol = Q.attend(q[rows], oc, np.array([0, adds[b]]), lens[b:b + 1], table[b:b + 1], 1, 100,
                                 np.zeros((adds[b], hd)))
            assert np.all(np.abs(got[rows] - want).max(axis=1) <= tol)
        if adds[1] > 1000:
            for i in (0, 1, 63, 99, 100, 4097, adds[1] // 2, adds[1] - 1):
                one = row0[1] + i
                # row i of a prompt that began at position 0 reads as one row of i + 1 tokens
                want, tol = Q.attend(q[one:one + 1], oc, np.array([0, 1]), [i + 1 + lens[1] - adds[1]], table[1:2], 1, 100,
                                     np.zeros((1, hd)))
                assert np.abs(got[one] - want[0]).max() <= tol[0], i
        dc.free()
