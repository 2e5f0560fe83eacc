"""Matrix products beside the factorizations: matrices in 8-bit floating point with a scale for each block of 128 (`quantize`, `product`,
`product_grads`), the orthogonal factor of a matrix by Newton-Schulz products (`orthogonalize`), and what the two are for next to a sweep:
`rangebasis`, an orthonormal basis of the leading directions of a large X.  The reference leaves such numerics to other packages.

The operators take and return torch tensors on the GPU; they run on torch's current stream of the tensors' device, do not wait, and can be
captured into a graph (a Quantized matrix used on another stream than its own needs what a tensor needs there: the streams ordered, the object kept).  `rangebasis` takes a numpy array like `execute` does, or a tensor."""
import ctypes as C
import functools
import math

import numpy as np

from . import _lib
from ._lib import ERR_BAD_ARG, NMFkError, _check

# (a, b, c) of X <- a X + (b S + c S S) X: steep at zero (a singular value grows 3.4445-fold a step), every singular value from about 0.0015
# to 1 is between 0.68 and 1.21 after five steps
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
# three more of the steps that converge (error^3 in each) make the columns orthonormal to 32 bits
CONVERGING = (1.875, -1.25, 0.375)

_TYPES = _U8 = _F8 = _F32 = _FORWARD = _TORCH = None


def _torch():
    """torch, imported when the first of these operators is called (the rest of the package does without)"""
    global _TYPES, _U8, _F8, _F32, _FORWARD, _TORCH
    if _TORCH is None:
        import torch

        _FORWARD = torch.autograd.forward_ad
        _TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
        _U8, _F8, _F32, _TORCH = torch.uint8, torch.float8_e4m3fn, torch.float32, torch
    return _TORCH


def _bad(msg):
    return NMFkError(ERR_BAD_ARG, msg)


def _no_derivative(x, name):
    if x.requires_grad and _TORCH.is_grad_enabled():
        raise _bad(f"{name} requires a gradient, which this operator does not record: pass {name}.detach()")
    if getattr(_FORWARD, "_current_level", 0) >= 0 and _FORWARD.unpack_dual(x).tangent is not None:
        raise _bad(f"{name} carries a forward-mode tangent, which this operator does not record: pass the primal of torch.autograd.forward_ad.unpack_dual({name})")


def _tensor(x, name, ndim=2):
    torch = _torch()
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise _bad(f"{name} must be a torch tensor on the GPU")
    if x.dtype not in _TYPES:
        raise _bad(f"{name} must be float32, bfloat16 or float16, not {x.dtype}")
    if ndim and x.dim() != ndim:
        raise _bad(f"{name} must be a matrix")
    _no_derivative(x, name)
    return x.resolve_neg() if x.is_neg() else x  # (is_neg: its entries are the negative of what its memory holds)


def _output(x, ndim=2):
    _tensor(x, "out", ndim)
    if x.is_neg():
        raise _bad("out must not be a view with a pending negation")
    return x


def _written(out):
    """tells autograd that a caller's tensor has changed, as torch's own in-place operations do"""
    if not out.is_inference():
        _TORCH.autograd.graph.increment_version(out)


def _stream(device):
    raw = getattr(_torch()._C, "_cuda_getCurrentRawStream", None)  # (a tenth of the time that a Stream object takes to make)
    return raw(device.index) if raw else _torch().cuda.current_stream(device).cuda_stream


@functools.lru_cache(4096)
def _product_workspace(m, n, k, t):
    nb = C.c_int64()
    _check(_lib.lib().nmfk_product_workspace(m, n, k, t, C.byref(nb)))
    return nb.value


@functools.lru_cache(4096)
def _grads_workspace(m, n, k, t):
    nb = C.c_int64()
    _check(_lib.lib().nmfk_product_grads_workspace(m, n, k, t, C.byref(nb)))
    return nb.value


@functools.lru_cache(4096)
def _orthogonalize_workspace(b, r, c):
    nb = C.c_int64()
    _check(_lib.lib().nmfk_orthogonalize_workspace(b, r, c, C.byref(nb)))
    return nb.value


@functools.lru_cache(64)
def _coefficients(key, steps):
    cf = np.asarray(key, dtype=np.float64)
    if cf.shape == (3,):
        cf = np.broadcast_to(cf, (steps, 3))
    if cf.shape != (steps, 3):
        raise _bad(f"coefficients must be (a, b, c) or {steps} such triples")
    cf = np.ascontiguousarray(cf)
    return cf, cf.ctypes.data


class Quantized:
    """A matrix in 8-bit floating point (e4m3) with a scale for each block of 128 entries of a row, or for each 128 x 128 tile.

    values   float8_e4m3fn (rows, cols)
    scales   float32 (rows, ceil(cols / 128)), tiles: (ceil(rows / 128), ceil(cols / 128))
    The matrix is values * scales.  Quantized(values, scales, tiles) takes a matrix quantized elsewhere and lays it out once, in whole blocks
    with the scales block by block (8192 x 8192: 24 us); what quantize() returns stands so already."""

    __slots__ = ("shape", "tiles", "device", "_buf", "_ldv", "_lds", "_pv", "_ps")

    def __init__(self, values, scales, tiles=False):
        torch = _torch()
        if not (isinstance(values, torch.Tensor) and isinstance(scales, torch.Tensor)) or values.device.type != "cuda" or scales.device != values.device:
            raise _bad("values and scales must be torch tensors on one GPU")
        if values.dtype not in (torch.float8_e4m3fn, torch.uint8) or values.dim() != 2 or scales.dtype != torch.float32:
            raise _bad("values must be a float8_e4m3fn matrix and scales float32")
        _no_derivative(values, "values")
        _no_derivative(scales, "scales")
        r, c = values.shape
        kb = -(-c // 128)
        if tuple(scales.shape) != ((-(-r // 128) if tiles else r), kb):
            raise _bad(f"{'tiles' if tiles else 'rows'} of a {r} x {c} matrix have {(-(-r // 128) if tiles else r)} x {kb} scales, not {tuple(scales.shape)}")
        self._make(r, c, bool(tiles), values.device)
        v = self._values()
        v[:, :c].copy_(values.view(torch.uint8))
        if c < self._ldv:
            v[:, c:].zero_()
        self.scales.copy_(scales.detach())

    def _make(self, r, c, tiles, device):
        # one allocation: r rows of whole blocks, then the scales block by block (kb x r, or kb x tiles)
        kb = -(-c // 128)
        self.shape, self.tiles, self.device = (r, c), tiles, device
        self._ldv, self._lds = kb * 128, -(-r // 128) if tiles else r
        self._buf = _TORCH.empty(r * self._ldv + 4 * kb * self._lds, dtype=_F8, device=device)
        self._pv = self._buf.data_ptr()
        self._ps = self._pv + r * self._ldv
        return self

    def _values(self):
        return self._buf.view(_U8).as_strided((self.shape[0], self._ldv), (self._ldv, 1))

    @property
    def values(self):
        r, c = self.shape
        return self._buf.as_strided((r, c), (self._ldv, 1))

    @property
    def scales(self):
        return self._buf.view(_F32).as_strided((self._lds, self._ldv // 128), (1, self._lds), self.shape[0] * self._ldv // 4)

    def dequantize(self, dtype=None):
        """the matrix that values and scales stand for (float32 unless told otherwise)"""
        s = self.scales.repeat_interleave(128, 1)[:, : self.shape[1]]
        if self.tiles:
            s = s.repeat_interleave(128, 0)[: self.shape[0]]
        return (self.values.float() * s).to(dtype or _F32)


def _contiguous_side(X):
    """X and its strides: as it is if its rows or its columns are contiguous, else a copy"""
    (r, c), (sr, sc) = X.shape, X.stride()
    if r == c == 1:  # (contiguous to torch whatever its strides)
        return X, 1, 1
    if not (sc == 1 and (sr >= c or r == 1)) and not (sr == 1 and (sc >= r or c == 1)):
        X = X.contiguous()
        sr, sc = X.stride()
    return X, sr, sc


def quantize(X, tiles=False, both=False):
    """X (a matrix of float32, bfloat16 or float16) in 8 bits with a scale for each block of 128 entries of a row, or (tiles) for each
    128 x 128 tile.  scale = max(max |x| / 448, 2^-126) over the block's finite entries, value = x / scale rounded to e4m3, ties to even; an
    entry that is not finite becomes NaN and leaves its block alone.
    both=True: a pair, X and its transpose (blocks along ITS rows), from one pass over X."""
    X = _tensor(X, "X")
    r, c = X.shape
    X, sr, sc = _contiguous_side(X)
    dev, tiles = X.device, bool(tiles)
    q = Quantized.__new__(Quantized)._make(r, c, tiles, dev)
    if not both:
        _check(_lib.lib().nmfk_quantize(dev.index, _stream(dev), _TYPES[X.dtype], X.data_ptr(), r, c, sr, sc, tiles, q._pv, q._ldv, q._ps, q._lds, None, 0, None, 0))
        return q
    t = Quantized.__new__(Quantized)._make(c, r, tiles, dev)
    _check(_lib.lib().nmfk_quantize(dev.index, _stream(dev), _TYPES[X.dtype], X.data_ptr(), r, c, sr, sc, tiles, q._pv, q._ldv, q._ps, q._lds, t._pv, t._ldv, t._ps, t._lds))
    return q, t


def _quantized(x, name):
    if not isinstance(x, Quantized):
        raise _bad(f"{name} must be a Quantized matrix (quantize)")
    return x


def product(A, B, dtype=None, out=None):
    """A * B' of two Quantized matrices (m x k and n x k), rounded once to dtype (float32, bfloat16 or float16).  float32: summed in 32 bits.
    The 16-bit types: by the 8-bit matrix instruction at twice the rate, which drops what lies more than 13 bits below the largest of 16 products it
    adds -- 1.4e-5 of the norm on normal entries, at most 2^-9 of the sum of an entry's |terms|.  Where large terms cancel and what they leave
    counts, take float32 and round the result.  The product of two blocks' scales is formed in 32 bits: below 2^-126 (entries of A times entries
    of B below about 2^-108) bits are lost, above 2^128 infinities or NaN come.
    out: the m x n tensor to write, rows contiguous."""
    torch = _torch()
    _quantized(A, "A")
    _quantized(B, "B")
    if A.shape[1] != B.shape[1] or A.device != B.device:
        raise _bad(f"A * B' needs rows of one length on one GPU, not {A.shape} on {A.device} and {B.shape} on {B.device}")
    (m, k), n, dev, given = A.shape, B.shape[0], A.device, out is not None
    if out is None:
        dtype = dtype or torch.float32
        if dtype not in _TYPES:
            raise _bad(f"dtype must be float32, bfloat16 or float16, not {dtype}")
        out = torch.empty((m, n), dtype=dtype, device=dev)
    else:
        _output(out)
        if tuple(out.shape) != (m, n) or out.device != dev or (dtype is not None and out.dtype != dtype) or (n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n):
            raise _bad(f"out must be {m} x {n} on {dev} with contiguous rows")
    t = _TYPES[out.dtype]
    nb = _product_workspace(m, n, k, t)
    work = torch.empty(nb, dtype=_U8, device=dev) if nb else None
    _check(_lib.lib().nmfk_product(dev.index, _stream(dev), m, n, k, A._pv, A._ldv, A._ps, A._lds, A.tiles, B._pv, B._ldv, B._ps, B._lds, B.tiles, t,
                                   out.data_ptr(), out.stride(0) if m > 1 else n, work.data_ptr() if nb else None, nb))
    if given:
        _written(out)
    return out


def product_grads(dY, At, Bt, dtype=None):
    """The backward pass of Y = product(A, B): (dA, dB) = (dY * B, dY' * A), both products in 8 bits.  dY and its transpose are quantized by
    rows; At and Bt are the Quantized transposes of A and of B (quantize(..., both=True) leaves them beside the forward's).  The gradients are
    those with respect to the matrices that the 8 bits stand for.  dtype (dY's own unless told otherwise) decides the arithmetic as in product."""
    torch = _torch()
    dY = _tensor(dY, "dY")
    _quantized(At, "At")
    _quantized(Bt, "Bt")
    m, n = dY.shape
    if At.shape[1] != m or Bt.shape[1] != n or At.shape[0] != Bt.shape[0] or At.device != dY.device or Bt.device != dY.device:
        raise _bad(f"dY {m} x {n} needs At k x {m} and Bt k x {n} on its GPU, not {At.shape} on {At.device} and {Bt.shape} on {Bt.device}")
    dtype = dtype or dY.dtype
    if dtype not in _TYPES:
        raise _bad(f"dtype must be float32, bfloat16 or float16, not {dtype}")
    dY, sr, sc = _contiguous_side(dY)
    k, dev, t = At.shape[0], dY.device, _TYPES[dtype]
    nb = _grads_workspace(m, n, k, t)
    dA, dB, work = torch.empty((m, k), dtype=dtype, device=dev), torch.empty((n, k), dtype=dtype, device=dev), torch.empty(nb, dtype=_U8, device=dev)
    _check(_lib.lib().nmfk_product_grads(dev.index, _stream(dev), m, n, k, _TYPES[dY.dtype], dY.data_ptr(), sr, sc, At._pv, At._ldv, At._ps, At._lds, At.tiles,
                                         Bt._pv, Bt._ldv, Bt._ps, Bt._lds, Bt.tiles, t, dA.data_ptr(), k, dB.data_ptr(), k, work.data_ptr(), nb))
    return dA, dB


def _extent(x):
    """first byte of a tensor and the one behind its last"""
    at = x.data_ptr()
    return at, at + (sum(st * (n - 1) for st, n in zip(x.stride(), x.shape)) + 1) * x.element_size()


def orthogonalize(G, steps=5, coefficients=None, out=None):
    """The orthogonal factor of G (..., rows, cols), or of each matrix of a stack, by Newton-Schulz products: X = G / |G|_F, then `steps`
    times X <- a X + (b S + c S S) X, S = X X' (of the transpose where rows > cols).  coefficients: (a, b, c), or one such triple per step.
    The default five steps bring every singular value from about 0.0015 |G|_F upwards to between 0.68 and 1.21, which is what an update wants;
    for orthonormal rows or columns add steps with (1.875, -1.25, 0.375).  Accuracy of fp32 in every step, or better, and one rounding to G's type:
    directions that G does not have come back as rounding noise, which grows like any small singular value.
    Zeros give zeros, an entry that is not finite gives NaN in its matrix.  out: where to write, G itself or apart from it."""
    torch = _torch()
    G = _tensor(G, "G", ndim=0)
    if G.dim() < 2:
        raise _bad("G must be a matrix or a stack of matrices")
    steps = int(steps)
    if steps < 1 or steps > 32:
        raise _bad("1 to 32 steps")
    if coefficients is None:
        key = COEFFICIENTS
    else:
        cf = np.asarray(coefficients, dtype=np.float64)
        key = tuple(cf.tolist()) if cf.ndim == 1 else tuple(map(tuple, cf.tolist())) if cf.ndim == 2 else ()
    cf, cf_at = _coefficients(key, steps)
    given = out is not None
    if out is None:
        if G.dim() > 3:
            g = G.reshape(math.prod(G.shape[:-2]), *G.shape[-2:])  # (a copy where the leading dimensions do not fold into one)
            return orthogonalize(g, steps, coefficients).view(G.shape)
        out = torch.empty_like(G)
    else:
        _output(out, ndim=0)
        if out.shape != G.shape or out.dtype != G.dtype or out.device != G.device:
            raise _bad("out must have G's shape, type and GPU")
        reach = 0  # of the dimensions with shorter strides
        for st, n in sorted((st, n) for st, n in zip(out.stride(), out.shape) if n > 1):
            if st <= reach:
                raise _bad("out must have a place for every entry, apart from the others")
            reach += st * (n - 1)
        if out.numel() and not (out.data_ptr() == G.data_ptr() and out.stride() == G.stride()):
            (a0, a1), (b0, b1) = _extent(out), _extent(G)
            if a0 < b1 and b0 < a1:
                raise _bad("out must be G itself or not overlap it")
    g, o = G, out
    if G.dim() == 2:
        (r, c), b = G.shape, 1
        gs, os = (0, *G.stride()), (0, *out.stride())
    else:
        if G.dim() > 3:
            try:
                o = out.view(math.prod(out.shape[:-2]), *out.shape[-2:])
            except RuntimeError:
                raise _bad("the leading dimensions of out must fold into one") from None
            g = o if out.data_ptr() == G.data_ptr() else G.reshape(o.shape)
        b, r, c = g.shape
        gs, os = g.stride(), o.stride()
    dev, nb = G.device, _orthogonalize_workspace(b, r, c)
    work = torch.empty(nb, dtype=_U8, device=dev) if nb else None
    _check(_lib.lib().nmfk_orthogonalize(dev.index, _stream(dev), _TYPES[G.dtype], b, r, c, g.data_ptr(), *gs, o.data_ptr(), *os,
                                         steps, cf_at, work.data_ptr() if nb else None, nb))
    if given:
        _written(out)
    return out


def rangebasis(X, k, oversample=8, iterations=2, seed=0, device=None):
    """An orthonormal basis of the k leading directions of X (n x m), by subspace iteration on X in 8 bits: products with X and X', each
    orthogonalized (65536 x 2048, k = 64: 3.6 ms).  Returns (Q, B, sigma): Q (n x k), B = Q' X (k x m, so X is near Q B), and sigma, the k leading singular values of X as the
    basis sees them.  Next to a sweep: sigma says where the candidate ranks end, Q and B are X compressed.  X is read once in 32 bits and kept in
    8, so sigma carries 8-bit noise: of about 3 % of |X| / sqrt(max(n, m)), below which nothing is resolved.
    Directions that X does not have (k above its rank) come back as noise of that size, or zero: their columns of Q are at most of length one.
    X: a numpy array (results are numpy arrays) or a torch tensor on the GPU (results are tensors).  NaN (missing data) is refused."""
    torch = _torch()
    host = not isinstance(X, torch.Tensor)
    if host:
        X = np.asarray(X)
        if X.ndim != 2:
            raise _bad("NMFk analysis can be executed for matrices!")
        if _lib.device_count() == 0:
            raise NMFkError(_lib.ERR_NO_DEVICE, "no usable gfx950 device: the library has no CPU fallback")
        X = torch.from_numpy(np.ascontiguousarray(X, dtype=np.float32)).to(torch.device("cuda", int(device or 0)))
    X = _tensor(X, "X")
    n, m = X.shape
    k = int(k)
    if not 1 <= k <= min(n, m):
        raise _bad(f"k must be between 1 and {min(n, m)}")
    low, high = (float(x) for x in torch.aminmax(X))
    top = max(-low, high)
    if not math.isfinite(top):
        raise _bad("X must be finite (no missing data)")
    e = math.frexp(top)[1]
    if abs(e) <= 40:
        e = 0
    else:  # far from 1: a copy by a power of two, so that neither the products nor the scales leave the range of fp32
        X = X.float() * 2.0 ** (-e // 2) * 2.0 ** (-e - -e // 2)
    r = min(k + max(0, int(oversample)), n, m)
    X8, Xt8 = quantize(X, tiles=True, both=True)
    g = torch.Generator(device=X.device)
    g.manual_seed(int(seed))
    steps = [COEFFICIENTS] * 10 + [CONVERGING] * 4

    def basis(y):
        return orthogonalize(y, len(steps), steps)

    Q = basis(product(X8, quantize(torch.randn(r, m, generator=g, device=X.device))))
    for _ in range(int(iterations)):
        Z = basis(product(Xt8, quantize(Q.t())))
        Q = basis(product(X8, quantize(Z.t())))
    B = (Q.t() @ X.float()).double()
    # the singular vectors of B from its r x r Gram matrix, in 64 bits: what the squares lose is below 1e-8 of the largest one, far below the noise of 8 bits
    # (an SVD of B itself does not converge on matrices of zeros)
    U = torch.linalg.eigh(B @ B.t())[1].flip(1)[:, :k]
    Q, B = (Q.double() @ U).float(), U.t() @ B * 2.0 ** e
    sigma, B = torch.linalg.vector_norm(B, dim=1).float(), B.float()
    return tuple(x.cpu().numpy() for x in (Q, B, sigma)) if host else (Q, B, sigma)
