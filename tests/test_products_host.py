"""CPU-only: the matrix operators (quantize, product, product_grads, orthogonalize, rangebasis) refuse what they cannot do before any GPU is
touched -- through the C ABI and through the Python entry points."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def NMFk():
    import nmfk_jl_amd

    nmfk_jl_amd.build()
    return nmfk_jl_amd


PTR = 1 << 20  # a plausible, aligned address: every call below is refused before it is used


def _last(L):
    return L.nmfk_last_error().decode()


QUANT = dict(device=0, stream=None, dtype=0, X=PTR, rows=300, cols=200, rs=200, cs=1, tiles=0, v=PTR, ldv=256, s=PTR, lds=300, tv=None, ldtv=0,
             ts=None, ldts=0)
QUANT_BAD = [dict(rows=-1), dict(dtype=3), dict(dtype=-1), dict(X=None), dict(v=None), dict(s=None), dict(rs=199), dict(rs=2, cs=2), dict(rs=0), dict(cs=0),
             dict(ldv=255), dict(ldv=240), dict(v=PTR + 8), dict(lds=299), dict(tv=PTR), dict(ts=PTR), dict(tv=PTR, ts=PTR, ldtv=256, ldts=200),
             dict(tv=PTR, ts=PTR, ldtv=384, ldts=199), dict(tv=PTR + 4, ts=PTR, ldtv=384, ldts=200), dict(rs=1, cs=299), dict(tiles=1, lds=2)]


@pytest.mark.parametrize("bad", QUANT_BAD, ids=str)
def test_quantize_refuses(NMFk, bad):
    L = NMFk.lib()
    assert L.nmfk_quantize(*{**QUANT, **bad}.values()) == 1, bad
    assert "nmfk_quantize" in _last(L)


def test_quantize_of_nothing_and_of_too_much(NMFk):
    L = NMFk.lib()
    assert L.nmfk_quantize(*{**QUANT, "rows": 0, "X": None, "v": None, "s": None}.values()) == 0
    assert L.nmfk_quantize(*{**QUANT, "rows": (1 << 22) + 1}.values()) == 6


PROD = dict(device=0, stream=None, m=10, n=20, k=200, A=PTR, lda=256, sA=PTR, ldsa=10, at=0, B=PTR, ldb=256, sB=PTR, ldsb=20, bt=0, dtype=0, Y=PTR, ldy=20,
            work=PTR, wb=1 << 40)
PROD_BAD = [dict(m=-1), dict(n=-3), dict(k=-1), dict(dtype=5), dict(A=None), dict(B=None), dict(sA=None), dict(sB=None), dict(Y=None), dict(ldy=19),
            dict(lda=255), dict(lda=128), dict(ldb=200), dict(A=PTR + 1), dict(B=PTR + 8), dict(ldsa=9), dict(ldsb=19), dict(at=1, ldsa=0)]


@pytest.mark.parametrize("bad", PROD_BAD, ids=str)
def test_product_refuses(NMFk, bad):
    L = NMFk.lib()
    assert L.nmfk_product(*{**PROD, **bad}.values()) == 1, bad
    assert "nmfk_product" in _last(L)


def test_product_of_nothing_sizes_and_workspace(NMFk):
    L = NMFk.lib()
    assert L.nmfk_product(*{**PROD, "m": 0}.values()) == 0
    assert L.nmfk_product(*{**PROD, "n": (1 << 22) + 1, "ldy": 1 << 23}.values()) == 6
    nb = C.c_int64()
    assert L.nmfk_product_workspace(10, 20, 0, 0, C.byref(nb)) == 0 and nb.value == 0
    assert L.nmfk_product_workspace(10, 20, -1, 0, C.byref(nb)) == 1
    assert L.nmfk_product_workspace(10, 20, 5, 0, None) == 1
    # a long sum of few outputs is split: the workspace is asked for, and a call without it refused
    assert L.nmfk_product_workspace(16, 64, 65536, 0, C.byref(nb)) == 0 and nb.value > 0
    big = {**PROD, "m": 16, "n": 64, "k": 65536, "lda": 65536, "ldb": 65536, "ldsa": 16, "ldsb": 64, "ldy": 64}
    for w in (dict(work=None), dict(wb=nb.value - 1), dict(work=PTR + 4)):
        assert L.nmfk_product(*{**big, **w}.values()) == 1
        assert "workspace" in _last(L)


GRADS = dict(device=0, stream=None, m=10, n=20, k=200, dt=0, dY=PTR, rs=20, cs=1, At=PTR, ldat=128, sAt=PTR, ldsat=200, att=0, Bt=PTR, ldbt=128, sBt=PTR, ldsbt=200,
             btt=0, dtype=0, dA=PTR, ldda=200, dB=PTR, lddb=200, work=PTR, wb=1 << 40)


@pytest.mark.parametrize("bad", [dict(m=-1), dict(n=-1), dict(k=-1), dict(dtype=7), dict(dt=7), dict(dY=None), dict(rs=3), dict(work=None), dict(wb=100), dict(work=PTR + 64)], ids=str)
def test_product_grads_refuses(NMFk, bad):
    L = NMFk.lib()
    assert L.nmfk_product_grads(*{**GRADS, **bad}.values()) == 1, bad
    assert "nmfk_" in _last(L)


def test_product_grads_of_nothing(NMFk):
    L = NMFk.lib()
    nb = C.c_int64()
    assert L.nmfk_product_grads_workspace(0, 0, 5, 0, C.byref(nb)) == 0 and nb.value == 0
    assert L.nmfk_product_grads_workspace(3, 4, 5, 0, None) == 1
    assert L.nmfk_product_grads(*{**GRADS, "m": 0, "n": 0, "work": None, "wb": 0}.values()) == 0


CF = (C.c_double * 15)(*([3.4445, -4.7750, 2.0315] * 5))
ORTHO = dict(device=0, stream=None, dtype=0, batch=2, rows=100, cols=20, G=PTR, gb=2000, gr=20, gc=1, O=PTR, ob=2000, orow=20, oc=1, steps=5,
             cf=C.addressof(CF), work=PTR, wb=1 << 40)


def _cf(*v):
    a = (C.c_double * len(v))(*v)
    return a, C.addressof(a)


@pytest.mark.parametrize("bad", [dict(batch=-1), dict(rows=-1), dict(cols=-2), dict(dtype=3), dict(steps=0), dict(steps=33), dict(cf=None), dict(G=None), dict(O=None),
                                 dict(work=None), dict(wb=16), dict(work=PTR + 16)], ids=str)
def test_orthogonalize_refuses(NMFk, bad):
    L = NMFk.lib()
    assert L.nmfk_orthogonalize(*{**ORTHO, **bad}.values()) == 1, bad
    assert "nmfk_orthogonalize" in _last(L)


@pytest.mark.parametrize("c", [(70.0, 0.0, 0.0), (float("nan"), 0, 0), (float("inf"), 0, 0), (1, 1e4, 0), (3.0, 10.0, 60.0)])
def test_orthogonalize_refuses_coefficients_that_blow_up(NMFk, c):
    keep, at = _cf(*c)
    assert NMFk.lib().nmfk_orthogonalize(*{**ORTHO, "steps": 1, "cf": at}.values()) == 1
    assert "coefficient" in _last(NMFk.lib())


def test_orthogonalize_of_nothing_and_of_too_much(NMFk):
    L = NMFk.lib()
    assert L.nmfk_orthogonalize(*{**ORTHO, "cols": 0}.values()) == 0
    nb = C.c_int64()
    assert L.nmfk_orthogonalize_workspace(1, 40000, 40000, C.byref(nb)) == 6
    assert L.nmfk_orthogonalize_workspace(1, 0, 5, C.byref(nb)) == 0 and nb.value == 0
    assert L.nmfk_orthogonalize_workspace(1, 5, 5, None) == 1
    for batch, rows, cols in ((1 << 22, 32768, 32768), (1 << 22, 64, 2048), (1 << 22, 1 << 22, 64)):  # nothing divides by zero on the way to the refusal
        assert L.nmfk_orthogonalize_workspace(batch, rows, cols, C.byref(nb)) == 6
    for batch, rows, cols in ((1 << 17, 1024, 2048), (256, 32768, 32768), (1, 1 << 22, 32768), (1 << 22, 256, 256), (1 << 22, 1, 1)):
        assert L.nmfk_orthogonalize_workspace(batch, rows, cols, C.byref(nb)) == 0 and nb.value > 0


def test_python_entry_points_refuse_what_is_not_on_the_gpu(NMFk):
    x = torch.ones(4, 4)
    for call in (lambda: NMFk.quantize(x), lambda: NMFk.quantize(np.ones((4, 4))), lambda: NMFk.orthogonalize(x), lambda: NMFk.product(x, x),
                 lambda: NMFk.product_grads(x, x, x), lambda: NMFk.Quantized(x, x), lambda: NMFk.rangebasis(x, 2)):
        with pytest.raises(NMFk.NMFkError) as e:
            call()
        assert e.value.code == 1


def test_rangebasis_has_no_cpu_fallback(NMFk):
    if NMFk.device_count() > 0:
        pytest.skip("a GPU is present")
    with pytest.raises(NMFk.NMFkError) as e:
        NMFk.rangebasis(np.ones((4, 4), np.float32), 2)
    assert e.value.code == 7
    with pytest.raises(NMFk.NMFkError) as e:
        NMFk.rangebasis(np.ones(4, np.float32), 2)
    assert e.value.code == 1
