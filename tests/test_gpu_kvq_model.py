"""Models over the paged 8-bit KV cache (vx_model_set_kv_pages) against the
oracle attending over the rows the GPU stored (its cache-store hook): decode,
verify and prompt batches on every forward path, roll-back into a page, the
context's end, speculative decoding, and what the option refuses and drops."""
import ctypes as C

import numpy as np
import pytest

import _kvq as Q
import _native as N
from _native import close, max_violation
from _oracle_model import OracleModel
from test_gpu_model import GpuModel, make

pytestmark = pytest.mark.gpu
O = N.oracle()


@pytest.fixture(scope="module")
def P():
    if not N.product_available():
        pytest.fail("product library not built")
    L = Q.bind(N.bind_vxh(N.product()))
    assert L.vxh_init() == 0, L.vxh_last_error()
    L.vx_model_set_kv_pages.argtypes = [C.POINTER(N.VxModelDev), C.c_int, C.c_int]
    return L


def options(P, mp, **over):
    opt = N.VxModelOptions()
    P.vx_model_get_options(mp, C.byref(opt))
    for k, v in over.items():
        setattr(opt, k, v)
    return P.vx_model_set_options(mp, C.byref(opt))


class Pair:
    """A GPU model on pages and an oracle that attends over the GPU's rows."""

    def __init__(self, P, tmp_path, seed, kind, page, hd, n_ctx=512, q4_kernel=0, cap=4096, h=4, kv=2, **over):
        path, raw, (self.L, self.d, self.h, self.kv, ff, self.V) = make(tmp_path, seed, L=2, d=h * hd, h=h, kv=kv,
                                                                       ff=2 * h * hd, V=500)
        self.P, self.n_ctx, self.kvd, self.hd, self.kind, self.page = P, n_ctx, kv * hd, hd, kind, page
        self.g = GpuModel(P, path, n_ctx=n_ctx, q4_kernel=q4_kernel, cap=cap)
        assert options(P, self.g.mp, ffn_gate_threshold=0.0, **over) == 0, N.product_error()
        assert P.vx_model_set_kv_pages(self.g.mp, kind, page) == 0, N.product_error()
        self.om = OracleModel(raw, self.L, self.d, h, kv, ff, self.V, n_ctx=n_ctx, q4_mode=q4_kernel, attn_cap=cap,
                              gate_thr=0.0)
        self.kc = self.om.k_cache.reshape(self.L, n_ctx, self.kvd)
        self.vc = self.om.v_cache.reshape(self.L, n_ctx, self.kvd)
        self.own = [np.zeros((self.L, self.kvd), np.float32) for _ in range(2)]
        self.om.m.kv_own_k, self.om.m.kv_own_v = (o.ctypes.data_as(C.c_void_p) for o in self.own)

    def rows(self, n):
        out = np.zeros((2, self.L, n, self.kvd), np.float32)
        for l in range(self.L):
            assert self.P.vx_model_read_kv(self.g.mp, l, n, out[0, l], out[1, l]) == 0, N.product_error()
        return out

    def check(self, got, toks, past, what, last_only=False):
        """got: the GPU's logits of toks at past..; the oracle's over the rows
        now in the cache, and its own rows against the stored ones."""
        n = min(past + len(toks), self.n_ctx)
        gpu = self.rows(n)
        self.kc[:, :n], self.vc[:, :n] = gpu
        self.om.m.kv_keep = 1
        row = np.zeros((1, self.V), np.float32)
        top = Q.TOP[self.kind]
        for j, t in enumerate(toks):
            p = min(past + j, n - 1)
            if last_only and j < len(toks) - 1 and j % 29:
                continue
            self.om.cache_len = past + j
            assert O.or_forward_all(self.om.ptr, np.array([t], np.int32), 1, row) == 0
            for own, w in zip(self.own, gpu):
                stored = w[:, p].reshape(self.L, -1, self.hd)
                mine = own.reshape(stored.shape)
                pg = p // self.page * self.page
                big = np.abs(w[:, pg:pg + self.page].reshape(self.L, -1, stored.shape[1], self.hd)).max(axis=(1, 3))
                scale = big[:, :, None] / top
                # rounded at most three times: as it came, and as its page's scale grew
                # twice; 2^-10 for the two sums' own fp32 rounding
                half = 0.5 * scale if self.kind == Q.INT8 else np.maximum(np.abs(mine) * 2.0 ** -4, scale * 2.0 ** -10)
                worst = (np.abs(stored - mine) - 3 * half - 2.0 ** -10 * scale * top).max()
                assert worst <= 0, (what, j, worst)
            if not last_only or j == len(toks) - 1:
                ref = row[0]
                mine = got[j] if not last_only else got
                assert close(mine, ref), (what, j, max_violation(mine, ref))

    def close(self):
        self.g.close()


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
@pytest.mark.parametrize("page,hd,over", [(32, 64, {}), (64, 128, {}), (128, 32, {}), (32, 96, {}),
                                          (32, 64, dict(fused=0)), (64, 64, dict(pro_max_rows=4))])
def test_decode_verify_and_prompt(P, tmp_path, kind, page, hd, over):
    """Token by token, verify batches of 1 to 16 rows after a roll-back, a
    prompt chunk on the large-M path, and decoding behind it."""
    print(f"paged model: type {kind}, page {page}, head_dim {hd}, {over}", flush=True)
    m = Pair(P, tmp_path, 700 + hd, kind, page, hd, **over)
    rng = np.random.default_rng(hd + kind)
    try:
        past = 0
        for M in [1, 1, 3, 1, 16, 2, 9, 31, 1, 5]:
            toks = rng.integers(0, m.V, M).astype(np.int32)
            got = np.concatenate([m.g.verify(toks[i:i + 16]) for i in range(0, M, 16)])
            if M <= 16:
                m.check(got, toks, past, f"{M} rows at {past}")
            past += M
            if M in (16, 9):
                past -= M - 2                       # refused drafts
                P.vx_model_kv_truncate(m.g.mp, past)
        prompt = rng.integers(0, m.V, 150).astype(np.int32)
        last = m.g.forward(prompt)                   # one large-M chunk
        m.check(last, prompt, past, "prompt", last_only=True)
        past += 150
        for M in (1, 4):
            toks = rng.integers(0, m.V, M).astype(np.int32)
            m.check(m.g.verify(toks), toks, past, f"{M} rows behind the prompt")
            past += M
        assert m.g.cache_len == past
    finally:
        m.close()


def test_x86_lanes(P, tmp_path):
    m = Pair(P, tmp_path, 31, Q.INT8, 32, 64, q4_kernel=1)
    rng = np.random.default_rng(2)
    try:
        past = 0
        for M in (5, 1, 16):
            toks = rng.integers(0, m.V, M).astype(np.int32)
            m.check(m.g.verify(toks), toks, past, f"{M} rows")
            past += M
    finally:
        m.close()


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
def test_end_of_the_context_and_cap(P, tmp_path, kind):
    """Tokens past the context take its last position; a cap on the attended
    positions; a prompt longer than the context."""
    m = Pair(P, tmp_path, 77, kind, 32, 64, n_ctx=75, cap=50)
    rng = np.random.default_rng(3)
    try:
        toks = rng.integers(0, m.V, 73).astype(np.int32)
        last = m.g.forward(toks)
        m.check(last, toks, 0, "prompt", last_only=True)
        toks = rng.integers(0, m.V, 2).astype(np.int32)
        m.check(m.g.verify(toks), toks, 73, "to the end")
        for i in range(3):
            toks = rng.integers(0, m.V, 1).astype(np.int32)
            m.check(m.g.verify(toks), toks, m.g.cache_len, f"past the end {i}")
            assert m.g.cache_len == 75
        P.vx_model_kv_truncate(m.g.mp, 0)
        toks = rng.integers(0, m.V, 130).astype(np.int32)
        m.g.forward(toks)
        assert m.g.cache_len == 75
    finally:
        m.close()


def test_switching_and_refusals(P, tmp_path):
    path, raw, (L, d, h, kv, ff, V) = make(tmp_path, 5, L=2, d=256, h=4, kv=2, ff=512, V=300)
    g = GpuModel(P, path, n_ctx=256)
    rng = np.random.default_rng(4)
    toks = rng.integers(0, V, 70).astype(np.int32)
    try:
        want = g.verify(toks)
        for bad in ((3, 32), (1, 16), (1, 0), (2, 48), (-1, 32)):
            assert P.vx_model_set_kv_pages(g.mp, *bad) == -3 or P.vx_model_set_kv_pages(g.mp, *bad) != 0
            assert g.cache_len == 70
        assert P.vx_model_set_kv_pages(None, 1, 32) != 0
        assert P.vx_model_set_kv_pages(g.mp, 0, 99) == 0 and g.cache_len == 70      # already so
        assert P.vx_model_set_kv_pages(g.mp, Q.INT8, 64) == 0, N.product_error()
        assert g.cache_len == 0 and not g.mp.contents.k_cache
        assert options(P, g.mp, kv_half=1) != 0
        a = g.verify(toks)
        assert g.mp.contents.k_cache
        assert np.abs(a - want).max() < 0.1 * np.abs(want).max()
        assert P.vx_model_set_kv_pages(g.mp, Q.INT8, 64) == 0 and g.cache_len == 70
        P.vx_model_kv_truncate(g.mp, 0)
        assert np.array_equal(g.verify(toks), a)                # the same calls, the same bits
        assert options(P, g.mp, attn_cap=33) == 0
        P.vx_model_kv_truncate(g.mp, 0)
        g.verify(toks)
        assert options(P, g.mp, attn_cap=4096) == 0
        assert P.vx_model_set_kv_pages(g.mp, Q.E4M3, 32) == 0 and g.cache_len == 0
        g.forward(toks)
        assert P.vx_model_set_kv_pages(g.mp, 0, 0) == 0 and g.cache_len == 0
        assert np.array_equal(g.verify(toks), want)
        assert options(P, g.mp, kv_half=1) == 0, N.product_error()
        assert P.vx_model_set_kv_pages(g.mp, Q.INT8, 32) != 0
        assert "kv_half" in N.product_error()
    finally:
        g.close()
    path, raw, sh = make(tmp_path, 6, L=1, d=128, h=8, kv=2, ff=256, V=100)           # head_dim 16
    g = GpuModel(P, path)
    try:
        assert P.vx_model_set_kv_pages(g.mp, Q.INT8, 32) != 0
        assert "head_dim" in N.product_error()
        g.verify(np.arange(3, dtype=np.int32))
    finally:
        g.close()


@pytest.mark.parametrize("kind", [Q.INT8, Q.E4M3])
def test_speculative_decoding(P, tmp_path, kind):
    """Both caches paged: greedy rounds end, agree with themselves, and a
    changed cache asks for a new prefill."""
    path, raw, (L, d, h, kv, ff, V) = make(tmp_path, 12, L=2, d=256, h=4, kv=2, ff=512, V=300)
    g, dr = GpuModel(P, path, n_ctx=256), GpuModel(P, path, n_ctx=256)
    st = P.vx_speculative_create(dr.mp, g.mp, 5)
    try:
        for mp in (g.mp, dr.mp):
            assert P.vx_model_set_kv_pages(mp, kind, 32) == 0
        P.vx_speculative_set_temp(st, 0.0, 1.0)
        prompt = np.random.default_rng(1).integers(0, V, 61).astype(np.int32)
        outs = []
        for _ in range(2):
            out = np.zeros(64, np.int32)
            assert P.vx_speculative_generate(st, prompt, len(prompt), out, 64) == 64, N.product_error()
            assert out.min() >= 0 and out.max() < V
            outs.append(out)
        assert np.array_equal(*outs)
        stats = N.VxSpecStats()
        P.vx_speculative_get_stats(st, C.byref(stats))
        # the draft is the target: only 8-bit rounding can part them
        assert stats.accepted > 0.5 * stats.drafted
        assert P.vx_model_set_kv_pages(g.mp, 0, 0) == 0
        out = np.zeros(8, np.int32)
        assert P.vx_speculative_decode(st, out, 8) == 0
        assert "prefill again" in N.product_error()
    finally:
        P.vx_speculative_destroy(st)
        g.close()
        dr.close()
