"""Workloads of the matrix-product operators that stand beside the factorizations: `quantize` (a matrix in 8-bit floating point with a
scale for each block of 128), `product` (A * B' of two such matrices), `product_grads` (the two products of its backward pass) and
`orthogonalize` (the orthogonal factor of a matrix, or of a stack of them, by Newton-Schulz products).

`own` selects what `run` computes: the plain form in elementary torch operations (False), or the calls a user makes of the package (True).

Definitions.
  quantize: a block is 128 consecutive entries of a row ("rows") or a 128 x 128 square ("tiles"); the last ones of a row or column may be
    shorter.  scale = max(max |x| of the block / 448, 2^-126) in 32 bits, value = x / scale (32 bits) rounded to e4m3, ties to even.
    With `both`, the transpose is quantized too, with blocks along ITS rows.
  product: Y[i, j] = sum_b sA[i, b] * sB[j, b] * sum_{t in block b} a[i, t] * b[j, t], rounded once to the output's type.
  product_grads of Y = A * B': dY and its transpose are quantized by rows; dA = dY8 * (B'8)', dB = dY'8 * (A'8)'.
  orthogonalize: X = G / |G|_F, then `steps` times X <- a X + (b S + c S S) X with S = X X' (rows no longer than columns; else its transpose).
"""
import math

import torch

own = False

COEF = (3.4445, -4.7750, 2.0315)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _package():
    import nmfk_jl_amd

    return nmfk_jl_amd


# ---- cases ----------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the data matrix of a large sweep (65536 x 2048), kept in 8 bits in both orientations: once per data set, the largest pass
        dict(name="quantize_data_both", op="quantize", rows=65536, cols=2048, tiles=True, both=True, type="f32"),
        # a block of activations on its way into a product: short, odd, a ragged last block
        dict(name="quantize_rows_ragged", op="quantize", rows=1025, cols=2000, tiles=False, both=False, type="bf16"),
        # one sample against a square map: a single row, where latency and the read of the map count
        dict(name="product_one_row", op="product", m=1, n=4096, k=4096, b_tiles=True, a_tiles=False, type="bf16"),
        # the data matrix times 64 directions: a tall matrix that is read once
        dict(name="product_data_64", op="product", m=65536, n=64, k=2048, b_tiles=False, a_tiles=True, type="f32"),
        # its transpose times 64 columns of length 65536: few outputs, a long sum
        dict(name="product_data_t_64", op="product", m=2048, n=64, k=65536, b_tiles=False, a_tiles=True, type="f32"),
        # a large square product: bound by the matrix pipes
        dict(name="product_square", op="product", m=8192, n=8192, k=8192, b_tiles=True, a_tiles=False, type="bf16"),
        # backward of an ordinary training step
        dict(name="grads_square", op="grads", m=4096, n=4096, k=4096, type="bf16"),
        # backward of a small step with odd sizes in every direction
        dict(name="grads_odd", op="grads", m=777, n=513, k=1111, type="f32"),
        # one factor W of the bench's data (8192 x 512 at k = 16): a latency-bound call
        dict(name="orthogonalize_factor", op="orthogonalize", batch=1, rows=8192, cols=16, spectrum="factor", steps=5, type="f32"),
        # the W of every restart of a sweep at once: 480 factors of 8192 x 16
        dict(name="orthogonalize_restarts", op="orthogonalize", batch=480, rows=8192, cols=16, spectrum="factor", steps=5, type="f32"),
        # the update of a square weight: bound by the matrix pipes
        dict(name="orthogonalize_square", op="orthogonalize", batch=1, rows=4096, cols=4096, spectrum="update", steps=5, type="f32"),
        # a stack of wide updates in 16 bits
        dict(name="orthogonalize_wide", op="orthogonalize", batch=4, rows=1000, cols=4096, spectrum="update", steps=5, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "grads", "orthogonalize", "orthogonalize"])
    t = rng.choice(["f32", "bf16", "f16"])
    if op == "quantize":
        rows = _log(rng, 1, 65536)
        cols = _log(rng, 1, min(8192, max(1, (1 << 27) // rows)))
        return dict(op=op, rows=rows, cols=cols, tiles=rng.random() < 0.5, both=rng.random() < 0.5, type=t)
    if op == "product":
        while True:
            m, n, k = _log(rng, 1, 65536), _log(rng, 1, 8192), _log(rng, 16, 65536)
            if m * k <= 1 << 27 and n * k <= 1 << 27 and m * n <= 1 << 26 and m * n * k <= 1 << 38:
                return dict(op=op, m=m, n=n, k=k, a_tiles=rng.random() < 0.5, b_tiles=rng.random() < 0.5, type=t)
    if op == "grads":
        while True:
            m, n, k = _log(rng, 16, 8192), _log(rng, 16, 8192), _log(rng, 16, 8192)
            if m * n * k <= 1 << 36:
                return dict(op=op, m=m, n=n, k=k, type=t)
    while True:
        small, ratio, batch = _log(rng, 1, 2048), rng.uniform(1, 12), _log(rng, 1, 480)
        if small <= 64:
            ratio = _log(rng, 1, 16384 // small)
        large = int(small * ratio)
        if batch * small * large <= 1 << 25 and batch * small * small * large <= 1 << 34:
            rows, cols = (small, large) if rng.random() < 0.5 else (large, small)
            return dict(op=op, batch=batch, rows=rows, cols=cols, spectrum=rng.choice(["factor", "update"]), steps=rng.choice([1, 3, 5, 6]), type=t)


# ---- inputs ---------------------------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _activations(g, rows, cols, dtype):
    """normal entries, with columns and rows of different size and a few outliers, as activations and gradients have"""
    x = _randn(g, rows, cols)
    x *= torch.exp(_randn(g, rows, 1) * 0.5) * torch.exp(_randn(g, 1, cols) * 0.7)
    return x.to(dtype)


def _plain_quantize(x, tiles):
    """(values as float8_e4m3fn [rows, cols], scales)"""
    x = x.float()
    r, c = x.shape
    br = 128 if tiles else 1
    nr, nc = -(-r // br), -(-c // 128)
    p = torch.zeros(nr * br, nc * 128, device=x.device, dtype=torch.float32)
    p[:r, :c] = x
    p = p.view(nr, br, nc, 128)
    top = p.abs().amax(dim=(1, 3))
    s = (top / torch.full_like(top, 448.0)).clamp_min(2.0 ** -126)  # (by a tensor: a division by a number is a product with its inverse)
    q = (p / s.view(nr, 1, nc, 1)).view(nr * br, nc * 128)[:r, :c].to(torch.float8_e4m3fn)
    return q.contiguous(), s


def _values(q, s, tiles, dtype=torch.float32):
    """the matrix that values and scales stand for"""
    if tiles:
        s = s.repeat_interleave(128, 0)[: q.shape[0]]
    return q.to(dtype) * s.to(dtype).repeat_interleave(128, 1)[:, : q.shape[1]]


def prepare(case, seed):
    g = _generator(seed)
    t = TYPES[case["type"]]
    op = case["op"]
    if op == "quantize":
        if case["tiles"] and case["type"] == "f32":  # a data matrix: nonnegative, with rows of different size
            x = torch.rand(case["rows"], case["cols"], generator=g, device="cuda") * torch.exp(_randn(g, case["rows"], 1))
        else:
            x = _activations(g, case["rows"], case["cols"], t)
        return dict(case=case, x=x)
    if op in ("product", "grads"):
        m, n, k = case["m"], case["n"], case["k"]
        a = _activations(g, m, k, t)
        b = _randn(g, n, k) / math.sqrt(k)
        if op == "product":
            parts = [_plain_quantize(a, case["a_tiles"]) + (case["a_tiles"],), _plain_quantize(b, case["b_tiles"]) + (case["b_tiles"],)]
            st = dict(case=case)
        else:  # what the forward pass left: the transposes of the activations (by rows) and of the weight (by tiles)
            parts = [_plain_quantize(a.t(), False) + (False,), _plain_quantize(b.t(), True) + (True,)]
            st = dict(case=case, dy=_activations(g, m, n, t) * 1e-3)
        st["parts"] = parts
        if own:
            st["handles"] = [_package().Quantized(q, s, tiles=tl) for q, s, tl in parts]
        return st
    shape = (case["batch"], case["rows"], case["cols"])
    if case["spectrum"] == "factor":  # nonnegative factors of a factorization
        x = torch.rand(shape, generator=g, device="cuda")
    else:  # an update: noise, and a few strong directions
        r = max(1, min(shape[1:]) // 16)
        x = _randn(g, *shape) + torch.bmm(_randn(g, shape[0], shape[1], r), _randn(g, shape[0], r, shape[2])) * 0.5
    return dict(case=case, x=x.to(t))


# ---- one pass ---------------------------------------------------------------------------------------------------------------

def _plain_orthogonalize(x, steps):
    t = x.dtype
    wide = x.shape[1] <= x.shape[2]
    x = x.float() if wide else x.float().mT.contiguous()
    n = x.double().square().sum(dim=(1, 2), keepdim=True).sqrt()
    x = torch.where(n > 0, x.double() / n, 0.0).float()
    a, b, c = COEF
    for _ in range(steps):
        s = torch.bmm(x, x.mT.contiguous())
        x = a * x + torch.bmm(b * s + c * torch.bmm(s, s), x)
    return (x if wide else x.mT).to(t)


def run(state):
    case = state["case"]
    op = case["op"]
    t = TYPES[case["type"]]
    if own:
        P = _package()
        if op == "quantize":
            q = P.quantize(state["x"], tiles=case["tiles"], both=case["both"])
            return [(h.values, h.scales) for h in (q if case["both"] else (q,))]
        if op == "product":
            return P.product(*state["handles"], dtype=t)
        if op == "grads":
            return P.product_grads(state["dy"], *state["handles"], dtype=t)
        return P.orthogonalize(state["x"], steps=case["steps"])
    if op == "quantize":
        x = state["x"]
        return [_plain_quantize(v, case["tiles"]) for v in ((x, x.t()) if case["both"] else (x,))]
    if op == "product":
        a, b = (_values(*p) for p in state["parts"])
        return (a @ b.t()).to(t)
    if op == "grads":
        at, bt = (_values(*p) for p in state["parts"])
        dy = _values(*_plain_quantize(state["dy"], False), False)
        dyt = _values(*_plain_quantize(state["dy"].t(), False), False)
        return (dy @ bt.t()).to(t), (dyt @ at.t()).to(t)
    return _plain_orthogonalize(state["x"], case["steps"])


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------

def _bytes8(r, c, tiles):
    return r * c + 4 * -(-c // 128) * (-(-r // 128) if tiles else r)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    op = case["op"]
    if op == "quantize":
        r, c = case["rows"], case["cols"]
        out = _bytes8(r, c, case["tiles"]) + (_bytes8(c, r, case["tiles"]) if case["both"] else 0)
        return dict(bytes=size * r * c + out, flops=2 * r * c)
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return dict(bytes=_bytes8(m, k, case["a_tiles"]) + _bytes8(n, k, case["b_tiles"]) + size * m * n, flops=2 * m * n * k)
    if op == "grads":
        m, n, k = case["m"], case["n"], case["k"]
        return dict(bytes=size * m * n + _bytes8(k, m, False) + _bytes8(k, n, True) + size * (m * k + n * k), flops=4 * m * n * k)
    s, l = sorted((case["rows"], case["cols"]))
    steps = case["steps"]
    # every product but the one onto X has a symmetric result: half its operations.  The least of: products onto X in every step; or one
    # Gram matrix, the polynomial of it step by step (square, two factors of the next one, the running product), one product onto X
    direct = steps * (s * s * l + s * s * s + 2 * s * s * l)
    gram = s * s * l + 2 * s * s * l + s ** 3 * (4 * steps - 3)
    return dict(bytes=2 * size * case["batch"] * s * l, flops=case["batch"] * min(direct, gram))


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------------

def _block_scales(x, tiles):
    """scales from the definition, per entry of x and per block"""
    r, c = x.shape
    rows = torch.arange(r, device=x.device) // (128 if tiles else 1)
    cols = torch.arange(c, device=x.device) // 128
    top = torch.zeros(int(rows[-1]) + 1, int(cols[-1]) + 1, device=x.device, dtype=torch.float64)
    flat = (rows[:, None] * top.shape[1] + cols[None, :]).reshape(-1)
    top.view(-1).scatter_reduce_(0, flat, x.double().abs().reshape(-1), "amax")
    return torch.clamp(top / 448.0, min=2.0 ** -126), flat


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        x = state["x"]
        return [(None, _block_scales(v, case["tiles"])[0]) for v in ((x, x.t()) if case["both"] else (x,))]
    d = torch.float64
    if op == "product":
        a, b = (_values(*p, dtype=d) for p in state["parts"])
        return a @ b.t()
    if op == "grads":
        at, bt = (_values(*p, dtype=d) for p in state["parts"])
        out = []
        for y, other in ((state["dy"], bt), (state["dy"].t(), at)):
            s, flat = _block_scales(y, False)
            s = s.float().double().view(-1)[flat].view(y.shape)
            v = (y.double() / s).float().to(torch.float8_e4m3fn).double() * s
            out.append(v @ other.t())
        return out
    a, b, c = COEF
    x = state["x"].double()
    flip = x.shape[1] > x.shape[2]
    if flip:
        x = x.mT
    out = torch.empty_like(x)
    for i in range(x.shape[0]):
        y = x[i] / torch.linalg.matrix_norm(x[i])
        for _ in range(case["steps"]):
            s = y @ y.t()
            y = a * y + b * (s @ y) + c * (s @ (s @ y))
        out[i] = y
    return out.mT if flip else out
