"""The matrix operators at the ends of what they accept: many steps and matrices of low rank, extreme norms, every size of tile, views and
outputs of unusual shape.

Tolerances of orthogonalize with a shorter side s <= 96.  u = 2^-24, e = 2^-53, f(t) = t (a + b t^2 + c t^4) a step on the singular values.
  S is formed and its polynomials are multiplied in 64 bits: S is off by (l + 2) e, each product of the iteration adds 3 s e, and an error of S
    reaches O through the derivative of the polynomial Q, at most A^2 for growth A = product of max |a + b t^2 + c t^4|.  4 A^2 e (l + 3 s steps) holds all of it.
  A growth of up to 512: Q is rounded to fp32 and applied in fp32, |error| <= (s + 3) u (|Q| |X|)[i, j].  Beyond: in 64 bits, and in groups of steps
    with a growth of up to 2048; between groups X is rounded to fp32, |error|_F <= u |X|_F, and a step takes an error of X to at most L = max |f'| of it
    (an odd function of a matrix has, in the Frobenius norm, the Lipschitz constant of the function).
  The result is rounded to fp32 and then to its type."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from test_gpu_products import CF, F8, HALF, P, TINY, TYPES, check_ortho, check_product, check_quantized, randn, ref_ortho, values64  # noqa: F401,E402

pytestmark = pytest.mark.gpu

CONVERGING = (1.875, -1.25, 0.375)
U, E = 2.0 ** -24, 2.0 ** -53


def step_bounds(cf, u):
    """growth, Lipschitz constant and largest singular value after a step on singular values up to u"""
    a, b, c = cf
    t = np.linspace(0.0, u, 100001)
    return (max(1.0, np.abs(a + b * t ** 2 + c * t ** 4).max()), np.abs(a + 3 * b * t ** 2 + 5 * c * t ** 4).max() * 1.0001,
            np.abs(a * t + b * t ** 3 + c * t ** 5).max() * 1.0001)


def short_reference(x, cf):
    """O of one matrix with rows <= columns in 64 bits, a bound of its entries' errors before the result is rounded, and the largest singular value"""
    s, l = x.shape
    n = torch.linalg.matrix_norm(x.double())
    x0 = y = torch.where(n > 0, x.double() / n, 0.0)
    q = torch.eye(s, dtype=torch.float64, device=x.device)
    u = growth = whole = 1.0
    tol = steps = 0
    for a, b, c in cf:
        g, lip, u_next = step_bounds((a, b, c), u)
        if steps and growth * g > 2048:
            tol += 4 * growth ** 2 * E * (l + 3 * s * steps) + U * float(y.norm())
            growth, steps = 1.0, 0
        growth, whole, steps, u = growth * g, whole * g, steps + 1, u_next
        sq = y @ y.t()
        p = b * sq + c * (sq @ sq)
        y, q = a * y + p @ y, a * q + p @ q
        tol = tol * lip
    tol += 4 * growth ** 2 * E * (l + 3 * s * steps)
    if whole <= 512:
        tol = tol + (s + 3) * U * (q.abs() @ x0.abs())
    return y, tol, u


def check_short(o, g, cf):
    assert o.shape == g.shape and o.dtype == g.dtype
    for x, y in zip(g.reshape(-1, *g.shape[-2:]), o.reshape(-1, *o.shape[-2:])):
        if x.shape[0] > x.shape[1]:
            x, y = x.t(), y.t()
        want, tol, top = short_reference(x, cf)
        assert bool(torch.isfinite(y).all())
        h = HALF[g.dtype]
        err = (y.double() - want).abs()
        bound = tol + (want.abs() + tol) * (U + h) * (1 + h) + TINY[g.dtype]
        assert bool((err <= bound).all()), f"largest error {float(err.max())}, largest error / tolerance {float((err / bound).max())}"
        assert float(torch.linalg.eigvalsh((y.double() @ y.double().t()).cpu())[-1]) ** 0.5 <= top * (1 + 8 * (h + U) * min(x.shape) ** 0.5)


def spectrum(name, s, l, seed=3):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *shape: torch.randn(*shape, generator=gen, dtype=torch.float64)
    if name == "rows twice":
        x = r(s, l)
        x = torch.cat([x[: (s + 1) // 2], x[: s // 2]])
    elif name == "low rank":
        k = max(1, s // 4)
        x = r(s, k) @ r(k, l)
    elif name == "ones":
        x = torch.ones(s, l, dtype=torch.float64)
    elif name == "binary":
        x = (torch.rand(s, 3, generator=gen) < 0.5).double() @ (torch.rand(3, l, generator=gen) < 0.5).double()
    elif name == "sizes":  # rows of very different size
        x = r(s, l) * torch.exp(2 * r(s, 1))
    else:  # condition
        q, w = torch.linalg.qr(r(s, s))[0], torch.linalg.qr(r(l, s))[0]
        x = (q * torch.logspace(0, -np.log10(float(name)), s, dtype=torch.float64)) @ w.t()
    return x.float().cuda()


SPECTRA = ["rows twice", "low rank", "ones", "binary", "sizes", "1e3", "1e6"]


# ---- orthogonalize, shorter side up to 96: its factor in 64 bits -------------------------------------------------------------------

@pytest.mark.parametrize("name", SPECTRA)
@pytest.mark.parametrize("s,l", [(2, 9), (16, 200), (17, 40), (40, 60), (48, 700), (64, 64), (65, 300), (80, 81), (96, 130)])
def test_short_side(P, name, s, l):
    for k in (1, 5, 6):
        g = spectrum(name, s, l)
        check_short(P.orthogonalize(g, steps=k), g, [CF] * k)
        g = g.t().contiguous()
        check_short(P.orthogonalize(g, steps=k), g, [CF] * k)
    for t in (torch.bfloat16, torch.float16):
        g = (spectrum(name, s, l) / 8).to(t)
        check_short(P.orthogonalize(g, steps=6), g, [CF] * 6)


@pytest.mark.parametrize("s", [1, 2, 16, 40, 90])
@pytest.mark.parametrize("size", [1e-36, 1e-39, 3e-45, 1e36, 3e38])
def test_short_side_of_any_norm(P, s, size):
    """matrices of low rank: null directions grow to 485 / |G|, which fp32 does not hold"""
    x = torch.zeros(s, 2 * s, device="cuda")
    x[0, 0] = size
    x[s // 2, 3 % (2 * s)] = size / 2
    check_short(P.orthogonalize(x), x, [CF] * 5)
    check_short(P.orthogonalize(x.t().contiguous()), x.t(), [CF] * 5)
    b = x.bfloat16()
    check_short(P.orthogonalize(b), b, [CF] * 5)
    g = spectrum("low rank", s, 3 * s)
    g = g / g.abs().max() * size
    check_short(P.orthogonalize(g), g, [CF] * 5)
    check_short(P.orthogonalize(g, steps=6), g, [CF] * 6)


# ---- orthogonalize, shorter side up to 96: many steps ----------------------------------------------------------------------------------

STEPS = {"7": [CF] * 7, "10": [CF] * 10, "14": [CF] * 14, "20": [CF] * 20, "32": [CF] * 32, "10 + 4": [CF] * 10 + [CONVERGING] * 4, "steep": [(100.0, -200.0, 101.0), (1 / 32, 0.0, 0.0)] + [CF] * 5,
         "24": [CF] * 8 + [CONVERGING] * 16}


@pytest.mark.parametrize("name", SPECTRA)
@pytest.mark.parametrize("steps", list(STEPS))
@pytest.mark.parametrize("s,l", [(1, 5), (16, 200), (24, 1100), (40, 60), (64, 70), (72, 130), (90, 300), (96, 96)])
def test_many_steps(P, name, steps, s, l):
    cf = STEPS[steps]
    g = spectrum(name, s, l)
    check_short(P.orthogonalize(g, len(cf), cf), g, cf)
    g = g.t().contiguous()
    check_short(P.orthogonalize(g, len(cf), cf), g, cf)
    for t in (torch.bfloat16, torch.float16):
        h = (g / 8).to(t)
        check_short(P.orthogonalize(h, len(cf), cf), h, cf)


@pytest.mark.parametrize("s,l", [(12, 3000), (40, 60), (72, 900), (96, 130)])
@pytest.mark.parametrize("name", ["sizes", "1e2", "1e3", "1e4"])
def test_many_steps_to_orthonormal(P, name, s, l):
    """ten default steps bring singular values from 2e-5 of the norm up, four that converge make the rows orthonormal: entries off by u of themselves
    give 2 u, what is left of the iteration and the 64 bits less than that"""
    g = spectrum(name, s, l)
    cf = [CF] * 10 + [CONVERGING] * 4
    o = P.orthogonalize(g, len(cf), cf).double()
    assert float((o @ o.t() - torch.eye(s, device="cuda")).abs().max()) <= 4 * U


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("shape", [(3, 20, 70), (2, 300, 40), (5, 96, 100), (260, 30, 64)])
def test_many_steps_in_place_and_strided(P, t, shape):
    cf = [CF] * 10 + [CONVERGING] * 4
    g = randn(31, *shape, t=TYPES[t])
    want = P.orthogonalize(g, len(cf), cf)
    check_short(want[-2:], g[-2:], cf)
    assert torch.equal(want, P.orthogonalize(g, len(cf), cf))
    out = torch.full((shape[0], shape[1] + 3, 2 * shape[2] + 5), 7.0, device="cuda", dtype=TYPES[t])
    view = out[:, 2:-1, 1:-4:2]
    P.orthogonalize(g, len(cf), cf, out=view)
    check_short(view[-2:], g[-2:], cf)
    view.fill_(7.0)
    assert bool((out == 7.0).all())
    inplace = g.clone()
    P.orthogonalize(inplace, len(cf), cf, out=inplace)
    assert torch.equal(inplace, want)
    turned = g.mT.contiguous().mT
    P.orthogonalize(turned, len(cf), cf, out=turned)
    check_short(turned[-2:], g[-2:], cf)


def test_many_steps_of_zeros_and_of_what_is_not_finite(P):
    for s in (3, 30, 90):
        for t in TYPES.values():
            g = randn(32, 5, s, 2 * s, t=t)
            g[1], g[2, 1, 2], g[3, 0, 0] = 0, float("nan"), float("-inf")
            o = P.orthogonalize(g, steps=20)
            assert bool((o[1] == 0).all()) and bool(torch.isnan(o[2]).all()) and bool(torch.isnan(o[3]).all())
            check_short(o[[0, 4]], g[[0, 4]], [CF] * 20)


def test_many_steps_of_large_stacks(P):
    """more than one launch of matrices, and more than one portion of a 16-bit stack"""
    for shape, t in (((40000, 3, 7), torch.float32), ((40000, 3, 7), torch.bfloat16), ((400, 90, 1000), torch.bfloat16), ((3, 60, 300000), torch.float16)):
        g = torch.randn(*shape, device="cuda").to(t)
        o = P.orthogonalize(g, steps=8)
        pick = sorted({0, 1, shape[0] // 2, shape[0] - 2, shape[0] - 1, min(32768, shape[0] - 1)})
        check_short(o[pick], g[pick], [CF] * 8)
        assert bool(torch.isfinite(o).all())


def test_many_steps_in_a_graph(P):
    g, h = randn(33, 4, 50, 90), randn(34, 2, 700, 16, t=torch.bfloat16)
    run = lambda: (P.orthogonalize(g, steps=12), P.orthogonalize(h, steps=12))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    cg = torch.cuda.CUDAGraph()
    with torch.cuda.graph(cg):
        out = run()
    for rep in range(4):
        for v in (g, h):
            v.copy_(torch.roll(v, 1, 0) * 1.25)
        want = run()
        for o in out:
            o.zero_()
        cg.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(out, want))


@pytest.mark.parametrize("kind", ["ones", "binary"])
def test_rangebasis_of_low_rank(P, kind):
    """a sketch of low rank: the singular values that X has come out, and their directions are orthonormal"""
    gen = torch.Generator().manual_seed(5)
    n, m, k = 600, 300, 4
    rank = 1 if kind == "ones" else 3
    X = torch.ones(n, m) if kind == "ones" else (torch.rand(n, 3, generator=gen) < 0.5).float() @ (torch.rand(3, m, generator=gen) < 0.5).float()
    want = torch.linalg.svdvals(X.double())
    Q, B, sigma = P.rangebasis(X.cuda(), k)
    # small whole numbers are exact in 8 bits up to the rounding of x / scale: 2^-4 of themselves at most, at random
    noise = 2.0 ** -4 * float(X.norm()) / m ** 0.5
    assert float((sigma.cpu().double() - want[:k]).abs().max()) <= noise
    lead = Q[:, :rank].double()
    assert float((lead.t() @ lead - torch.eye(rank, device="cuda")).abs().max()) <= 1e-5
    assert float(torch.linalg.matrix_norm(Q.double(), 2)) <= 1 + 1e-5
    assert float((Q.double() @ B.double() - X.cuda().double()).norm()) <= noise * k ** 0.5


# ---- views and outputs of unusual shape -------------------------------------------------------------------------------------------------

def test_orthogonalize_stacks_whose_leading_dimensions_do_not_fold(P):
    for s, l in ((20, 40), (100, 130)):
        g = randn(41, 2, 3, s, l).permute(1, 0, 2, 3)
        o = P.orthogonalize(g)
        assert o.shape == g.shape
        check_ortho(o, g)
        g = randn(42, 2, 3, 2, l, s).permute(2, 0, 1, 4, 3)
        check_ortho(P.orthogonalize(g), g)
        with pytest.raises(P.NMFkError, match="fold"):
            P.orthogonalize(g, out=torch.empty_like(g))
    g = randn(43, 2, 3, 5, 7)
    assert P.orthogonalize(g).stride() == g.stride() and P.orthogonalize(g.mT).stride() == g.mT.stride()
    for shape in ((2, 3, 0, 5), (0, 2, 3, 5), (2, 0, 4, 4)):
        e = torch.empty(shape, device="cuda")
        assert P.orthogonalize(e).shape == shape and P.orthogonalize(e, out=torch.empty_like(e)).shape == shape




# ---- quantize, views of one entry ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("tiles", [False, True])
def test_quantize_one_entry_of_a_larger_matrix(P, tiles):
    x = randn(44, 5, 9)
    for v in (x[2:3, 4:5], x[:1, ::3][:, :1], x.t()[3:4, ::5][:, :1], x[:1, 1:2].expand(1, 1), x[::5, ::9]):
        q, w = P.quantize(v, tiles=tiles, both=True)
        check_quantized(q, v, tiles)
        check_quantized(w, v.t(), tiles)
        check_quantized(P.quantize(v, tiles=tiles), v, tiles)
    v = x[::5, ::9]
    da, db = P.product_grads(v, P.quantize(randn(47, 30, 1)), P.quantize(randn(48, 30, 1)))
    assert da.shape == db.shape == (1, 30)


# ---- tensors that stand for something else than their memory ------------------------------------------------------------------------------

def test_views_with_a_pending_negation(P):
    """the imaginary part of a conjugate: torch keeps the sign apart from the memory"""
    z = torch.complex(randn(51, 40, 300), randn(52, 40, 300))
    v = z.conj().imag
    assert v.is_neg()
    plain = v.clone()
    assert not plain.is_neg()
    for tiles in (False, True):
        check_quantized(P.quantize(v, tiles=tiles), plain, tiles)
    assert torch.equal(P.orthogonalize(v), P.orthogonalize(plain))
    at, bt = P.quantize(randn(53, 20, 40)), P.quantize(randn(54, 20, 300))
    for got, want in zip(P.product_grads(v, at, bt), P.product_grads(plain, at, bt)):
        assert torch.equal(got, want)
    for f in (lambda: P.orthogonalize(plain, out=v), lambda: P.orthogonalize(v, out=v), lambda: P.product(P.quantize(randn(55, 40, 64)), P.quantize(randn(56, 300, 64)), out=v)):
        with pytest.raises(P.NMFkError, match="negat"):
            f()


def test_forward_mode_tangents_are_refused(P):
    """no operator records a tangent: it must not vanish without a word"""
    import torch.autograd.forward_ad as fwAD

    x, w = randn(57, 6, 8), P.quantize(randn(58, 5, 8))
    at, bt = P.quantize(randn(59, 4, 6)), P.quantize(randn(60, 4, 8))
    with fwAD.dual_level():
        d = fwAD.make_dual(x, torch.ones_like(x))
        for f in (lambda: P.quantize(d), lambda: P.orthogonalize(d), lambda: P.product_grads(d, at, bt), lambda: P.rangebasis(d, 2),
                  lambda: P.orthogonalize(x, out=d), lambda: P.product(P.quantize(x), P.quantize(randn(61, 8, 8)), out=d)):
            with pytest.raises(P.NMFkError, match="tangent"):
                f()
        P.quantize(x), P.orthogonalize(x)  # a tensor without one is taken inside a level, too
        P.quantize(fwAD.unpack_dual(d).primal)


def test_quantized_refuses_a_gradient_it_does_not_record(P):
    import torch.autograd.forward_ad as fwAD

    v, s = P.quantize(randn(62, 6, 200)).values, torch.ones(6, 2, device="cuda", requires_grad=True)
    with pytest.raises(P.NMFkError, match="detach"):
        P.Quantized(v, s)
    P.Quantized(v, s.detach())
    with torch.no_grad():
        q = P.Quantized(v, s)
    assert not q.scales.requires_grad
    with fwAD.dual_level():
        with pytest.raises(P.NMFkError, match="tangent"):
            P.Quantized(v, fwAD.make_dual(s.detach(), torch.ones_like(s)))


def test_outputs_whose_entries_share_memory_are_refused(P):
    base = torch.zeros(1000, device="cuda")
    g = randn(63, 5, 8)
    for shape, strides in (((5, 8), (1, 1)), ((5, 8), (4, 1)), ((5, 8), (1, 3)), ((3, 5, 8), (8, 8, 1)), ((3, 5, 8), (39, 8, 1)), ((2, 3, 5, 8), (40, 40, 8, 1)), ((5, 8), (0, 1)),
                           ((3, 5, 8), (7, 35, 1))):
        out = base.as_strided(shape, strides)
        with pytest.raises(P.NMFkError, match="place for every entry"):
            P.orthogonalize(g.expand(shape).contiguous(), out=out)
        with pytest.raises(P.NMFkError, match="place for every entry"):
            P.orthogonalize(out, out=out)
    for shape, strides in (((5, 8), (8, 1)), ((5, 8), (1, 5)), ((5, 8), (20, 2)), ((3, 5, 8), (8, 24, 1)), ((3, 5, 8), (1, 24, 3)), ((1, 5, 8), (0, 8, 1)), ((5, 1), (1, 0)), ((3, 1, 8), (16, 16, 2))):
        out = base.as_strided(shape, strides)
        gg = randn(64, *shape)
        assert P.orthogonalize(gg, out=out) is out
        check_ortho(out, gg)


def test_writing_out_is_a_change_that_autograd_sees(P):
    x = torch.ones(6, 8, device="cuda", requires_grad=True)
    a, b = P.quantize(randn(65, 6, 40)), P.quantize(randn(66, 8, 40))
    for write in (lambda w: P.orthogonalize(w, out=w), lambda w: P.orthogonalize(randn(67, 6, 8), out=w), lambda w: P.product(a, b, out=w)):
        w = randn(68, 6, 8)
        y = (x * w).sum()
        write(w)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        w = randn(69, 6, 8)
        P.orthogonalize(w, out=w)
        P.product(a, b, out=w)
    P.product(a, b, out=w)
    leaf = torch.ones(6, 8, device="cuda", requires_grad=True)
    with torch.no_grad():
        P.product(a, b, out=leaf)
        P.orthogonalize(leaf, out=leaf)
    (leaf * 2).sum().backward()


# ---- sizes beyond what one launch holds -------------------------------------------------------------------------------------------------

def test_quantize_rows_of_more_blocks_than_a_launch_holds(P):
    """4194304 x 4100 of bf16 (34 GB): 138 million blocks of a row, 32 threads each"""
    r, c = 1 << 22, 4100
    x = torch.zeros(r, c, dtype=torch.bfloat16, device="cuda")
    at = [0, 1, 1000003, 2033600, 2033601, 2033602, r // 2, r - 2, r - 1]
    rows = randn(71, len(at), c, t=torch.bfloat16)
    x[at] = rows
    q = P.quantize(x)
    assert q.shape == (r, c)
    got, want = q.values[at], P.quantize(rows)
    assert torch.equal(got.view(torch.uint8), want.values.view(torch.uint8))
    assert torch.equal(q.scales[at], want.scales)
    s = q.scales
    assert int((s != 2.0 ** -126).sum()) == int((want.scales != 2.0 ** -126).sum())  # every other block: zeros
    del x
    v = q._values()
    for i in range(0, r, 1 << 20):  # (a part at a time: a reduction of bytes takes eight times their memory)
        assert int((v[i:i + (1 << 20)] != 0).sum()) == int((want._values()[[k for k, a in enumerate(at) if i <= a < i + (1 << 20)]] != 0).sum())


def test_product_of_no_terms_with_many_outputs(P):
    """k = 0 gives zeros, also where the outputs are more than the threads that a launch holds"""
    m, n = 65537, 65600
    a, b = P.quantize(torch.empty(m, 0, device="cuda")), P.quantize(torch.empty(n, 0, device="cuda"))
    out = torch.full((m, n + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    y = P.product(a, b, out=out[:, :n])
    assert int(torch.count_nonzero(y)) == 0
    assert bool((out[:, n:] == 7.0).all())


# ---- every kernel of the large forms ------------------------------------------------------------------------------------------------------
# Which tiles a size takes is a matter of an estimate; with the one of today: (sides of the Gram matrix, its square, the product onto X; "split": some of
# the sums are)

@pytest.mark.parametrize("shape,t", [
    ((2000, 2100), "f32"),     # 128 split, 128 split, 128
    ((2050, 2150), "f16"),     # the same, one entry more than whole tiles
    ((4, 1000, 4096), "bf16"),  # 128 split, 128, 128
    ((2, 1501, 1500), "f32"),  # 128, 128, 128
    ((4096, 4109), "f32"),     # 128: a whole round and a split rest; 128
    ((4090, 4095), "f32"),     # 128: a whole round and a split rest; 256
    ((6200, 2500), "bf16"),    # 128, 128, 256
    ((3000, 3001), "f32"),     # 64: a whole round and a split rest; 128
    ((1500, 6000), "f16"),     # 128 split
    ((16000, 700), "f32"),     # 64 split; 128
    ((16, 513, 520), "bf16"),  # 64; 128
    ((97, 16384), "f32"),      # 64 in 64 parts
])
def test_orthogonalize_tiles(P, shape, t):
    g = randn(81, *shape, t=TYPES[t])
    o = P.orthogonalize(g, steps=3)
    check_ortho(o, g, 3)
    assert torch.equal(o, P.orthogonalize(g, steps=3))


def test_orthogonalize_large_layouts_of_large_tiles(P):
    """128 and 256 tiles with the turned layout, an output apart from its surroundings, and in place"""
    for s, l in ((1500, 1600), (3900, 4090)):
        g = randn(82, l, s).t()
        o = P.orthogonalize(g, steps=2)
        check_ortho(o, g, 2)
        out = torch.full((s + 3, l + 9), 5.0, device="cuda")
        P.orthogonalize(g, steps=2, out=out[1:s + 1, 4:l + 4])
        check_ortho(out[1:s + 1, 4:l + 4], g, 2)
        out[1:s + 1, 4:l + 4] = 5.0
        assert bool((out == 5.0).all())
        inplace = g.clone()
        P.orthogonalize(inplace, steps=2, out=inplace)
        check_ortho(inplace, g, 2)


@pytest.mark.parametrize("s", [97, 130])
def test_orthogonalize_more_matrices_than_a_launch_of_the_large_form(P, s):
    """32768 matrices a launch: the second launch's places in the workspace, and its matrices"""
    g = torch.randn(32768 + 70, s, s + 1, device="cuda", dtype=torch.bfloat16)
    g[32768 + 3] = 0
    o = P.orthogonalize(g, steps=2)
    pick = [0, 1, 32766, 32767, 32768, 32769, 32768 + 3, 32768 + 69]
    check_ortho(o[[p for p in pick if p != 32768 + 3]], g[[p for p in pick if p != 32768 + 3]], 2)
    assert bool((o[32768 + 3] == 0).all())
    each = P.orthogonalize(g[32768:], steps=2)
    assert float((each.float() - o[32768:].float()).abs().max()) <= 2.0 ** -7 * float(each.float().abs().max())


def test_orthogonalize_far_offsets_of_the_large_form(P):
    """100 rows of 4098 entries, 4095 apart: the last one more than 2^30 entries from the first, the last matrix more than 2^32 bytes"""
    big = torch.empty(2, 100, 1 << 24, device="cuda")
    big.uniform_(-1, 1)
    v = big[:, :, ::4095]
    o = P.orthogonalize(v, steps=2)
    check_ortho(o, v, 2)
    P.orthogonalize(v, steps=2, out=v)
    assert torch.equal(v, o) or float((v - o).abs().max()) <= 2.0 ** -18
    w = big[:, :, 1 << 20::5].mT[:, :2000]  # columns of 100, 2^24 entries apart, rows 5 apart
    check_ortho(P.orthogonalize(w, steps=2), w, 2)


@pytest.mark.parametrize("steps", [14, 20, 32])
@pytest.mark.parametrize("s,l", [(100, 130), (160, 900), (1200, 1300)])
def test_large_form_with_many_steps_stays_bounded(P, steps, s, l):
    """directions that G does not have come back as rounding noise, never beyond the largest value of the steps"""
    g = spectrum("low rank", s, l)
    o = P.orthogonalize(g, steps=steps).double()
    assert bool(torch.isfinite(o).all())
    top = torch.linalg.eigvalsh((o @ o.t()).cpu())
    assert float(top[-1]) ** 0.5 <= 1.21
    u, sv, _ = torch.linalg.svd(g.double().cpu(), full_matrices=False)
    u = u[:, sv > 1e-3 * sv[0]].cuda()
    lead = torch.linalg.svdvals((u.t() @ o).cpu())
    assert float(lead[-1]) >= 0.65  # what is there comes to between 0.68 and 1.21


@pytest.mark.parametrize("m,n,k", [(2048, 2048, 256), (8192, 8192, 128), (4000, 4100, 300), (3500, 3400, 1000), (20, 9000, 700), (50, 8200, 500), (64, 30000, 130), (40, 8192, 129), (64, 65, 9000)])
@pytest.mark.parametrize("ta,tb", [(False, True), (False, False), (True, True), (True, False)])
def test_product_tiles(P, m, n, k, ta, tb):
    """256 x 256, 128 x 128 and the forms of up to 64 rows with 16 and 32 columns a workgroup"""
    a, b = P.quantize(randn(m + k, m, k), tiles=ta), P.quantize(randn(n * 3 + k, n, k), tiles=tb)
    for t in TYPES.values():
        check_product(P.product(a, b, dtype=t), values64(a), values64(b), t)


# ---- what the type of a product's result decides ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("m", [3, 200])
def test_product_where_large_terms_cancel(P, m):
    """448^2 - 448^2 and fourteen terms of 8 in one group of sixteen: fp32 results hold the small ones, 16-bit ones are within 2^-9 of the sum of |terms|"""
    a, b = torch.zeros(m, 128, device="cuda"), torch.zeros(70, 128, device="cuda")
    a[:, 0], a[:, 1], a[:, 2:16] = 448.0, -448.0, 2.0
    b[:, 0], b[:, 1], b[:, 2:16] = 448.0, 448.0, 4.0
    qa, qb = P.quantize(a), P.quantize(b)
    assert float(qa.scales.min()) == float(qa.scales.max()) == 1.0
    mag = 2 * 448.0 ** 2 + 14 * 8
    y = P.product(qa, qb).double()
    assert bool(((y - 112).abs() <= (256 + 2 + 3) * U * mag).all())
    for t in (torch.bfloat16, torch.float16):
        y = P.product(qa, qb, dtype=t).double()
        assert bool(((y - 112).abs() <= 2.0 ** -9 * mag).all())
        exact = P.product(qa, qb).to(t).double()  # as documented: fp32, rounded by the caller
        assert bool(((exact - 112).abs() <= (256 + 2 + 3) * U * mag + HALF[t] * 128).all())
    # the same of the backward pass: dA = dY8 * (B'8)'
    da, _ = P.product_grads(a[:, :70].contiguous(), P.quantize(torch.zeros(5, m, device="cuda")), P.quantize(b[:5, :70].contiguous()), dtype=torch.float32)
    assert bool(((da.double() - 112).abs() <= (256 + 2 + 3) * U * mag).all())


# ---- rangebasis: matrices without, or of few, directions, and of any size -----------------------------------------------------------------

@pytest.mark.parametrize("n,m,k", [(300, 120, 8), (3000, 1200, 88), (200, 120, 100), (1, 50, 1), (700, 1, 1), (1, 1, 1)])
@pytest.mark.parametrize("kind", ["zeros", "one entry", "ones"])
def test_rangebasis_of_few_directions(P, n, m, k, kind):
    X = torch.ones(n, m, device="cuda") if kind == "ones" else torch.zeros(n, m, device="cuda")
    if kind == "one entry":
        X[n // 2, m // 3] = -3.0
    Q, B, sigma = P.rangebasis(X, k)
    top = {"zeros": 0.0, "one entry": 3.0, "ones": (n * m) ** 0.5}[kind]
    assert Q.shape == (n, k) and B.shape == (k, m) and bool(torch.isfinite(Q).all()) and bool(torch.isfinite(B).all())
    assert abs(float(sigma[0]) - top) <= 1e-5 * top
    assert float(sigma[1:].sum()) <= 2.0 ** -4 * k * top
    assert float((Q.double() @ B.double() - X.double()).norm()) <= 1e-4 * top


@pytest.mark.parametrize("e", [-125, -100, -45, 45, 100, 119])
def test_rangebasis_of_any_size(P, e):
    """scaling X by a power of two scales B and sigma, and changes no bit of Q"""
    gen = torch.Generator().manual_seed(9)
    X = (torch.rand(400, 3, generator=gen) @ torch.rand(3, 250, generator=gen) + 0.01 * torch.rand(400, 250, generator=gen)).cuda()
    X[X < 2.0 ** -8] = 2.0 ** -8  # (no entry becomes subnormal at 2^-125 but for its last bits)
    X = (X * 2.0 ** 14).round() * 2.0 ** -14
    if e == 119:
        X = X[:20, :10].contiguous()  # its singular values fit into fp32
    Q, B, sigma = P.rangebasis(X, 4)
    scaled = X * 2.0 ** (e // 2) * 2.0 ** (e - e // 2)
    for t in (torch.float32, torch.bfloat16) if e > -125 else (torch.float32,):  # (bf16 has no room for the last bits at 2^-125)
        x, y = (X, scaled) if t == torch.float32 else (X.to(t), (X.to(t).float() * 2.0 ** (e // 2) * 2.0 ** (e - e // 2)).to(t))
        (q0, b0, s0), (q1, b1, s1) = P.rangebasis(x, 4), P.rangebasis(y, 4)
        back = lambda v: v.double() * 2.0 ** -e
        assert torch.equal(q0, q1)
        assert float((back(s1) - s0.double()).abs().max()) <= 2.0 ** -20 * float(s0[0])
        assert float((back(b1) - b0.double()).abs().max()) <= 2.0 ** -20 * float(s0[0])
    assert float((scaled.double() - Q.double() @ B.double() * 2.0 ** e).norm()) <= 2.0 ** e * 2.0 ** -4 * float(X.norm())


@pytest.mark.parametrize("size", [3e38, 1e38, 2.0 ** -126, 2.0 ** -149])
@pytest.mark.parametrize("r,c", [(1, 1), (2, 2), (40, 30)])
def test_rangebasis_of_the_largest_and_smallest_entries(P, size, r, c):
    X = torch.zeros(r, c, device="cuda")
    X[0, 0] = -size
    X[-1, -1] = size
    rank = 1 if r == c == 1 else 2
    Q, B, sigma = P.rangebasis(X, rank)
    want = float(X[-1, -1])
    assert float((sigma.double() - want).abs().max()) <= 1e-5 * want
    # (an entry of B is rounded to a multiple of 2^-149: off by 2^-150 at most, `rank` of them in an entry of Q B)
    assert float((Q.double() @ B.double() - X.double()).abs().max()) <= 1e-4 * want + rank * 2.0 ** -150


# ---- errors that are not the call's own ---------------------------------------------------------------------------------------------------

def test_an_error_left_by_another_call_is_not_reported(P):
    """a refused call of the HIP runtime (here: a device that does not exist) leaves its error behind for whoever asks next"""
    import ctypes as C

    path = {line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line}
    hip = C.CDLL(path.pop())
    x, g, h = randn(91, 40, 300), randn(92, 20, 40), randn(93, 120, 130)
    want = (P.quantize(x), P.orthogonalize(g), P.orthogonalize(h))
    q = want[0]
    y = P.product(q, q)
    torch.cuda.synchronize()
    for f, w in ((lambda: P.quantize(x).values.view(torch.uint8), want[0].values.view(torch.uint8)), (lambda: P.orthogonalize(g), want[1]), (lambda: P.orthogonalize(h), want[2]),
                 (lambda: P.product(q, q), y)):
        assert hip.hipSetDevice(12345) != 0
        got = f()
        hip.hipGetLastError()
        assert torch.equal(got, w)
