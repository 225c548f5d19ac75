"""Paged 8-bit KV cache, without a GPU: the handle's layout, the refusals of
every entry point (arguments are checked before anything is launched), what a
model on pages allocates and gives back, and the numpy oracle's codes against
their definition."""
import ctypes as C
import glob
import os
import re
import subprocess

import numpy as np
import pytest

import _kvq as Q
import _native as N


@pytest.fixture(scope="module")
def P():
    if not N.product_available():
        pytest.fail("product library not built (run __graft_entry__.build())")
    return Q.bind(N.product())


def test_handle_mirror_matches_the_header(tmp_path):
    names = [n for n, _ in Q.Kvq._fields_]
    src = ['#include <stdio.h>', '#include <stddef.h>', '#include "vxh.h"', "int main(void) {",
           'printf("%zu\\n", sizeof(vxh_kvq));']
    src += [f'printf("%zu\\n", offsetof(vxh_kvq, {n}));' for n in names] + ["return 0; }"]
    c = tmp_path / "a.c"
    c.write_text("\n".join(src) + "\n")
    subprocess.run(["gcc", "-std=gnu11", "-I", os.path.join(N.REPO, "include"), str(c), "-o", str(tmp_path / "a")],
                   check=True)
    out = [int(x) for x in subprocess.run([str(tmp_path / "a")], check=True, capture_output=True,
                                          text=True).stdout.split()]
    assert out == [C.sizeof(Q.Kvq)] + [getattr(Q.Kvq, n).offset for n in names]


PTR = C.c_void_p(1 << 20)       # never followed: the calls below are refused
MIS = C.c_void_p((1 << 20) + 4)


def handle(**over):
    c = Q.Kvq(type=1, page=32, n_pages=8, n_kv_heads=2, head_dim=64, k=1 << 20, v=1 << 20, ks=1 << 20, vs=1 << 20)
    for n, v in over.items():
        setattr(c, n, v)
    return c


BAD_HANDLES = [dict(type=0), dict(type=3), dict(page=16), dict(page=48), dict(page=256), dict(head_dim=48),
               dict(head_dim=160), dict(head_dim=0), dict(n_kv_heads=0), dict(n_pages=0), dict(k=None), dict(vs=None),
               dict(n_pages=1 << 26)]


@pytest.mark.parametrize("over", BAD_HANDLES)
def test_bad_handles_are_refused_everywhere(P, over):
    c = C.byref(handle(**over))
    ws = Q.Workspace(part=1 << 20, part_floats=1 << 40)
    assert P.vxh_kvq_write(c, PTR, 128, PTR, 128, PTR, 4, None) == -3
    assert P.vxh_kvq_read(c, PTR, 4, PTR, 128, PTR, 128, None) == -3
    assert P.vxh_attention_kvq(PTR, 128, PTR, PTR, 1, 1, 1, PTR, 4, 2, c, 0, PTR, 128, C.byref(ws), None) == -3
    assert P.vxh_last_error()


@pytest.mark.parametrize("args", [(0, 32, 8, 2, 64), (1, 33, 8, 2, 64), (1, 32, 0, 2, 64), (1, 32, 8, 0, 64),
                                  (1, 32, 8, 2, 40), (2, 128, 1 << 24, 2, 64), (1, 32, -1, 2, 64)])
def test_alloc_refuses(P, args):
    c = Q.Kvq(k=5)
    assert P.vxh_kvq_alloc(C.byref(c), *args) == -3
    assert c.k is None and c.vs is None
    assert P.vxh_kvq_free(C.byref(c)) == 0      # nothing to free
    assert P.vxh_kvq_alloc(None, 1, 32, 8, 2, 64) == -3
    assert P.vxh_kvq_free(None) == 0


@pytest.mark.parametrize("k,ldk,v,ldv,slot,R", [
    (None, 128, PTR, 128, PTR, 4), (PTR, 128, None, 128, PTR, 4), (PTR, 128, PTR, 128, None, 4),
    (PTR, 124, PTR, 128, PTR, 4), (PTR, 128, PTR, 100, PTR, 4), (PTR, 130, PTR, 128, PTR, 4),
    (PTR, 128, PTR, 129, PTR, 4), (MIS, 128, PTR, 128, PTR, 4), (PTR, 128, MIS, 128, PTR, 4),
    (PTR, 128, PTR, 128, PTR, 0), (PTR, 128, PTR, 128, PTR, -1), (PTR, 128, PTR, 128, PTR, 8193)])
def test_rows_refused(P, k, ldk, v, ldv, slot, R):
    c = C.byref(handle())
    assert P.vxh_kvq_write(c, k, ldk, v, ldv, slot, R, None) == -3
    assert P.vxh_kvq_read(c, slot, R, k, ldk, v, ldv, None) == -3


def tables_args(**over):
    a = dict(len=PTR, add=C.c_void_p(2 << 20), n=4, page=32, free=PTR, n_free=4, table=PTR, ld=8,
             len_out=C.c_void_p(3 << 20), row0=PTR, pos=PTR, slot=PTR, max_rows=16, counts=PTR)
    a.update(over)
    return list(a.values()) + [None]


@pytest.mark.parametrize("over", [
    dict(len=None), dict(add=None), dict(free=None), dict(table=None), dict(len_out=None), dict(row0=None),
    dict(pos=None), dict(slot=None), dict(counts=None), dict(n=0), dict(n=4097), dict(page=16), dict(page=31),
    dict(n_free=-1), dict(ld=0), dict(max_rows=0), dict(max_rows=(1 << 18) + 1), dict(len_out=PTR),
    dict(len_out=C.c_void_p((1 << 20) + 12)), dict(len_out=C.c_void_p((2 << 20) - 8))])
def test_tables_refuse(P, over):
    assert P.vxh_page_tables(*tables_args(**over)) == -3
    assert b"page_tables" in P.vxh_last_error()


def attend_args(**over):
    a = dict(q=PTR, ldq=256, row0=PTR, len=PTR, n=2, rows=4, seq_rows=2, table=PTR, ld=8, heads=4, c=C.byref(handle()),
             cap=0, out=PTR, ld_out=256, ws=C.byref(Q.Workspace(part=1 << 20, part_floats=1 << 40)))
    a.update(over)
    return list(a.values()) + [None]


@pytest.mark.parametrize("over", [
    dict(q=None), dict(row0=None), dict(len=None), dict(table=None), dict(out=None), dict(ws=None), dict(n=0),
    dict(n=4097), dict(rows=0), dict(rows=(1 << 18) + 1), dict(seq_rows=0), dict(ld=0), dict(heads=0), dict(heads=3),
    dict(heads=-2), dict(cap=-1), dict(ldq=252), dict(ldq=257), dict(ld_out=252), dict(ld_out=258), dict(q=MIS),
    dict(out=MIS), dict(c=None)])
def test_attention_refuses(P, over):
    assert P.vxh_attention_kvq(*attend_args(**over)) == -3
    assert b"attention_kvq" in P.vxh_last_error()


@pytest.mark.parametrize("over", [dict(k=(1 << 20) + 4), dict(v=(1 << 20) + 8), dict(ks=(1 << 20) + 2),
                                  dict(vs=(1 << 20) + 1), dict(n_kv_heads=1 << 26)])
def test_handles_of_arrays_that_cannot_be_loaded(P, over):
    """Arrays off their alignment, and heads whose row passes 32 bits."""
    c = C.byref(handle(**over))
    ws = Q.Workspace(acc=1 << 20, part=1 << 20, part_floats=1 << 40)
    big = 0x7FFFFFFC
    assert P.vxh_kvq_write(c, PTR, big, PTR, big, PTR, 4, None) == -3
    assert P.vxh_kvq_read(c, PTR, 4, PTR, big, PTR, big, None) == -3
    assert P.vxh_attention_kvq(PTR, big, PTR, PTR, 1, 1, 1, PTR, 4, 1 << 26, c, 0, PTR, big, C.byref(ws), None) == -3


def test_counts_that_pass_32_bits_are_refused(P):
    ws = C.byref(Q.Workspace(acc=1 << 20, part=1 << 20, part_floats=1 << 40))
    big = 0x7FFFFFFC
    for heads, rows in ((1 << 26, 1), (1 << 25, 1), (1 << 24, 128), (8192, 1 << 18)):
        assert P.vxh_attention_kvq(*attend_args(heads=heads, rows=rows, ldq=big, ld_out=big, ws=ws)) == -3
    assert P.vxh_page_tables(*tables_args(page=128, ld=1 << 24)) == -3
    assert P.vxh_page_tables(*tables_args(page=32, ld=1 << 26)) == -3


def test_oracle_codes_are_the_nearest():
    """nearest() against a search over every code."""
    rng = np.random.default_rng(5)
    y = np.concatenate([rng.normal(0, 60, 3000), rng.normal(0, 1, 1000), [0, 0.5, 1.5, -2.5, 126.5, 127.5, 1e4, -1e4]])
    for kind, vals in ((Q.INT8, np.arange(-127.0, 128)), (Q.E4M3, Q.E4M3_VALUES[np.isfinite(Q.E4M3_VALUES)])):
        got = Q.nearest(y, kind)
        d = np.abs(y[:, None] - vals[None, :]).min(axis=1)
        assert np.array_equal(np.abs(got - y), d)
    assert Q.nearest(np.array([0.5, 1.5, 2.5, -0.5]), Q.INT8).tolist() == [0, 2, 2, -0.0]
    # e4m3 steps of 1/4 between 2 and 4: ties go to the even mantissa
    assert Q.nearest(np.array([2.125, 2.375, 2.0 ** -10, 3 * 2.0 ** -10]), Q.E4M3).tolist() == [2.0, 2.5, 0.0, 2.0 ** -8]


# --------------------------------------------------------------------------
# a model's memory: host/*.c over a stand-in device layer that counts
# --------------------------------------------------------------------------
@pytest.fixture(scope="module")
def H(tmp_path_factory):
    from test_prefill_buffers import BODIES, PRELUDE
    d = tmp_path_factory.mktemp("host")
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(N.REPO, "include", "vxh.h")).read(), flags=re.S)
    bodies = dict(BODIES)
    bodies["vxh_kvq_alloc"] = """memset(c, 0, sizeof *c);
    if (vxh_malloc(&c->k, 1000)) return VXH_ERR_ALLOC;
    if (vxh_malloc(&c->v, 1000)) { vxh_free(c->k); memset(c, 0, sizeof *c); return VXH_ERR_ALLOC; }
    return 0;"""
    bodies["vxh_kvq_free"] = "vxh_free(c->k); vxh_free(c->v); memset(c, 0, sizeof *c); return 0;"
    src = PRELUDE
    for ret, name, args in re.findall(r"^(int|size_t|void|const char \*) ?(vxh_\w+)\(([^;]*)\);", text, flags=re.M):
        src += "%s %s(%s) { %s }\n" % (ret, name, args, bodies.pop(name, "" if ret == "void" else "return 0;"))
    assert not bodies, sorted(bodies)
    (d / "stub.c").write_text(src)
    so = str(d / "host.so")
    subprocess.run(["gcc", "-std=gnu11", "-O1", "-shared", "-fPIC", "-I", os.path.join(N.REPO, "include"), "-o", so,
                    str(d / "stub.c")] + sorted(glob.glob(os.path.join(N.REPO, "veltrix-engine_amd", "host", "*.c"))) +
                   ["-lm", "-Wl,-z,defs"], check=True)
    L = C.CDLL(so)
    L.vx_model_create_synthetic.argtypes = [C.POINTER(N.VxModelConfig), C.POINTER(N.VxSynthSpec),
                                            C.POINTER(C.POINTER(N.VxModelDev))]
    L.vx_model_set_kv_pages.argtypes = [C.POINTER(N.VxModelDev), C.c_int, C.c_int]
    L.vx_model_forward.argtypes = [C.POINTER(N.VxModelDev), N.i32p, C.c_int, N.f32p]
    L.vx_model_destroy.argtypes = [C.POINTER(N.VxModelDev)]
    return L


def test_a_paged_model_returns_its_memory(H):
    budget, used = (C.c_size_t.in_dll(H, n) for n in ("st_budget", "st_used"))
    cfg = N.VxModelConfig()
    cfg.n_layers, cfg.n_heads, cfg.n_kv_heads, cfg.n_embd = 3, 2, 2, 128
    cfg.n_ff, cfg.n_vocab, cfg.n_ctx = 256, 64, 1000
    spec = N.VxSynthSpec(seed=1, std=0.02, matrix_type=2, embd_type=2, output_type=2)
    lg = np.zeros(64, np.float32)

    def walk():
        """Every kind of cache in turn; the return codes of the forwards."""
        m = C.POINTER(N.VxModelDev)()
        rc = [H.vx_model_create_synthetic(C.byref(cfg), C.byref(spec), C.byref(m))]
        if rc[0] == 0:
            for kind, n in ((1, 5), (0, 60), (2, 70), (1, 1), (1, 60)):
                assert H.vx_model_set_kv_pages(m, kind, 32) == 0
                rc.append(H.vx_model_forward(m, np.zeros(n, np.int32), n, lg))
            H.vx_model_destroy(m)
        return rc

    budget.value = 1 << 40
    start = used.value
    assert walk() == [0] * 6
    assert used.value == start
    # and when memory ends anywhere on the way
    m = C.POINTER(N.VxModelDev)()
    assert H.vx_model_create_synthetic(C.byref(cfg), C.byref(spec), C.byref(m)) == 0
    model = used.value - start
    H.vx_model_destroy(m)
    failed = 0
    for extra in range(0, 3_000_000, 1500):
        budget.value = start + model + extra
        failed += any(walk())
        assert used.value == start, extra
    assert failed > 100
