"""The microscaled 4-bit (MXFP4) operators as measured work: quantisation, product, linear layer, training step.

MXFP4 holds 32 consecutive elements of a row in 4 bits each (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and
their negatives) next to one power of two (an e8m0 byte). ``run`` computes each operator either in
elementary 32-bit torch operations (``own`` false) or through ``gpumon.ops.mx`` (``own`` true).

Row-major parts of a quantised matrix of ``rows`` x ``k``, as both sides take them: ``codes``
[rows, ceil(k/32)*16] uint8 (the even element in the low nibble) and ``scales`` [rows, ceil(k/32)]
uint8 (the exponent + 127).
"""

import math

import torch

own = False

BLOCK = 32
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
MAX_PRODUCT = 8192 ** 3  # the largest listed product, in multiply-adds


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # quantisation, there and back ("axis" 1: blocks along a row; 0: down a column; "both": as a
        # training step needs its operands, the two of them from one reading)
        # one token's activations of a 8192-wide layer: the latency of a call
        {"name": "quantize_token", "op": "quantize", "rows": 1, "k": 8192, "axis": "1", "dtype": "bf16"},
        # the activations of a long prompt
        {"name": "quantize_prompt", "op": "quantize", "rows": 8192, "k": 8192, "axis": "1", "dtype": "bf16"},
        # a master weight in 32 bits on the way to its training operands, odd in both sizes
        {"name": "quantize_both_odd", "op": "quantize", "rows": 4099, "k": 2053, "axis": "both", "dtype": "f32"},
        # products of two quantised matrices
        # the two sizes of this repository's matrix-product tenants
        {"name": "matmul_4096", "op": "matmul", "m": 4096, "n": 4096, "k": 4096, "dtype": "bf16"},
        {"name": "matmul_8192", "op": "matmul", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16"},
        # a ragged batch on a layer with odd sizes, sums handed on in 32 bits
        {"name": "matmul_odd", "op": "matmul", "m": 777, "n": 1411, "k": 2999, "dtype": "f32"},
        # linear layer on weights quantised beforehand (serving)
        # one token: a decode step of one sequence
        {"name": "linear_1", "op": "linear", "m": 1, "n": 8192, "k": 8192, "dtype": "bf16"},
        # a small decode batch on a layer of odd sizes
        {"name": "linear_13_odd", "op": "linear", "m": 13, "n": 7001, "k": 5005, "dtype": "f16"},
        # a larger decode batch
        {"name": "linear_64", "op": "linear", "m": 64, "n": 8192, "k": 8192, "dtype": "bf16"},
        # a prompt's chunk
        {"name": "linear_2048", "op": "linear", "m": 2048, "n": 8192, "k": 4096, "dtype": "bf16"},
        # training step of a linear layer: output, input gradient and weight gradient
        {"name": "train_4096", "op": "train", "m": 4096, "n": 4096, "k": 8192, "dtype": "bf16"},
        # a short packed batch with odd sizes
        {"name": "train_odd", "op": "train", "m": 613, "n": 1000, "k": 1337, "dtype": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "linear", "train"])
    if op == "quantize":
        rows, k = _log(rng, 1, 16384), _log(rng, 1, 16384)
        rows = max(1, min(rows, 8192 * 8192 // k))
        return {"op": op, "rows": rows, "k": k, "axis": rng.choice(["1", "0", "both"]),
                "dtype": rng.choice(["bf16", "f16", "f32"])}
    if op == "linear":
        # half of them decode batches
        m = _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 64, 4096)
        n, k = _log(rng, 64, 16384), _log(rng, 64, 16384)
    elif op == "matmul":
        m, n, k = _log(rng, 1, 16384), _log(rng, 16, 16384), _log(rng, 16, 16384)
    else:
        m, n, k = _log(rng, 1, 8192), _log(rng, 32, 8192), _log(rng, 32, 8192)
    if op == "train":
        m = max(1, min(m, 4096 * 4096 * 8192 // (n * k)))
    m = max(1, min(m, MAX_PRODUCT // (n * k)))
    return {"op": op, "m": m, "n": n, "k": k, "dtype": rng.choice(["bf16", "f16", "f32"] if op == "matmul" else ["bf16", "f16"])}


def work(case):
    s = SIZE[case["dtype"]]
    mx = 0.5 + 1.0 / BLOCK  # bytes of a quantised element
    if case["op"] == "quantize":
        n = case["rows"] * case["k"]
        copies = 2 if case["axis"] == "both" else 1
        return {"bytes": n * s * (1 + copies), "flops": 4 * n * copies}
    m, n, k = case["m"], case["n"], case["k"]
    if case["op"] == "matmul":
        return {"bytes": int((m + n) * k * mx) + m * n * s, "flops": 2 * m * n * k}
    if case["op"] == "linear":
        return {"bytes": m * k * s + int(n * k * mx) + m * n * s, "flops": 2 * m * n * k}
    return {"bytes": 2 * s * (m * k + n * k + m * n), "flops": 6 * m * n * k}


# ------------------------------------------------------------------------------------ inputs
def _activations(g, rows, k, dtype):
    """Normal values with a few channels that run far larger than the rest, and empty rows of a padded batch."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    x *= 1.0 + 30.0 * (torch.rand(k, generator=g, device="cuda") > 0.995)
    x *= torch.rand(rows, 1, generator=g, device="cuda") > 0.01 * (rows > 1)
    return x.to(dtype)


def _weights(g, n, k, dtype):
    return (torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)).to(dtype)


def _gradients(g, m, n, dtype):
    """Gradients differ in size from token to token by orders of magnitude."""
    d = torch.randn(m, n, generator=g, device="cuda")
    return (d * torch.exp(2.0 * torch.randn(m, 1, generator=g, device="cuda")) * 1e-2).to(dtype)


def _pack(index, scale):
    """Nibbles [rows, blocks, 32] and scale bytes [rows, blocks] to the row-major parts."""
    rows, blocks, _ = index.shape
    return (index[:, :, 0::2] | (index[:, :, 1::2] << 4)).reshape(rows, blocks * 16), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = {"case": case, "dtype": dt}
    op = case["op"]
    if op == "quantize":
        st["x"] = _activations(g, case["rows"], case["k"], dt)
        return st
    m, n, k = case["m"], case["n"], case["k"]
    st["x"] = _activations(g, m, k, torch.bfloat16 if op == "matmul" else dt)
    w = _weights(g, n, k, torch.bfloat16 if op == "matmul" else dt)
    if op == "train":
        st["w"] = w
        st["dy"] = _gradients(g, m, n, dt)
        return st
    st["w"] = _pack(*_encode(w))
    if op == "matmul":
        st["x"] = _pack(*_encode(st["x"]))
    if own:
        from gpumon.ops import mx

        st["w_mx"] = mx.MxTensor.pack(*st["w"], k)
        if op == "matmul":
            st["x_mx"] = mx.MxTensor.pack(*st["x"], k)
    return st


# ------------------------------------------------------------------------------------ plain form
def _pow2(e):
    """2^e in 32 bits for whole numbers e of normal range, from the bits."""
    return ((e + 127) << 23).view(torch.float32)


def _blocks(x):
    rows, k = x.shape
    pad = -k % BLOCK
    x = x.float()
    if pad:
        x = torch.cat([x, x.new_zeros(rows, pad)], 1)
    return x.view(rows, -1, BLOCK)


def _encode(x):
    """Nibbles and scale bytes of x, blocks along its last axis."""
    b = _blocks(x)
    amax = b.abs().amax(2)
    # frexp: amax = f * 2^e with f in [0.5, 1), so floor(log2 amax) = e - 1; the largest element is 6 = 1.5 * 2^2
    e = (torch.frexp(amax).exponent.to(torch.int32) - 3).clamp(-127, 125)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    # times 2^-e in two exact steps, since 2^127 is the largest power of two of the type
    h = torch.div(-e, 2, rounding_mode="floor")
    a = (b.abs() * _pow2(h).unsqueeze(2)) * _pow2(-e - h).unsqueeze(2)
    # halfway points between neighbours, and which of them go up: those whose upper neighbour's code is even
    q = (a > 0.25).to(torch.uint8)
    for up, border in ((1, 0.75), (0, 1.25), (1, 1.75), (0, 2.5), (1, 3.5), (0, 5.0)):
        q += (a >= border) if up else (a > border)
    bad = ~torch.isfinite(b).all(2)
    q = q | (torch.signbit(b).to(torch.uint8) << 3)
    q = torch.where(bad.unsqueeze(2), torch.zeros_like(q), q)
    return q, torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _values(q, scale, k):
    """What nibbles and scale bytes stand for, in 32 bits, [rows, k]."""
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), device=q.device)
    e = scale.to(torch.int32) - 127
    h = torch.div(e, 2, rounding_mode="floor")
    v = grid[q.long()] * _pow2(h).unsqueeze(2) * _pow2(e - h).unsqueeze(2)
    v = torch.where((scale == 255).unsqueeze(2), torch.full_like(v, float("nan")), v)
    return v.reshape(q.shape[0], -1)[:, :k]


def _rounded(x):
    """x as MXFP4 holds it, in 32 bits."""
    return _values(*_encode(x), x.shape[1])


def _unpack(parts, k):
    codes, scale = parts
    q = torch.stack([codes & 15, codes >> 4], 2).reshape(codes.shape[0], -1, BLOCK)
    return _values(q, scale, k)


def _plain(st):
    case, dt = st["case"], st["dtype"]
    op, k = case["op"], case["k"]
    x = st["x"]
    if op == "quantize":
        out = []
        if case["axis"] in ("1", "both"):
            out.append(_rounded(x).to(dt))
        if case["axis"] in ("0", "both"):
            out.append(_rounded(x.t()).to(dt))
        return out
    if op == "matmul":
        return (_unpack(x, k) @ _unpack(st["w"], k).t()).to(dt)
    if op == "linear":
        return (_rounded(x) @ _unpack(st["w"], k).t()).to(dt)
    w, dy = st["w"], st["dy"]
    y = _rounded(x) @ _rounded(w).t()
    dx = _rounded(dy) @ _rounded(w.t()).t()
    dw = _rounded(dy.t()) @ _rounded(x.t()).t()
    return [y.to(dt), dx.to(dt), dw.to(dt)]


def run(state):
    if not own:
        return _plain(state)
    from gpumon.ops import mx

    case, dt, x = state["case"], state["dtype"], state["x"]
    op = case["op"]
    if op == "quantize":
        if case["axis"] == "both":
            qs = mx.quantize_both(x)
        else:
            qs = [mx.quantize(x, axis=int(case["axis"]))]
        return [mx.dequantize(q, dt) for q in qs]  # "0": the rows of the result are x's columns
    if op == "matmul":
        return mx.matmul(state["x_mx"], state["w_mx"], dt)
    if op == "linear":
        return mx.linear(x, state["w_mx"])
    y, saved = mx.linear_train(x, state["w"])
    dx, dw = mx.linear_grad(state["dy"], saved)
    return [y, dx, dw]


# ------------------------------------------------------------------------------------ in 64 bits
def _unit(e):
    return e.to(torch.int64).add(1023).bitwise_left_shift(52).view(torch.float64)


def _exact_round(x):
    """MXFP4 of x from the definition: the grid's spacing at |t| is half the power of two below it, at least 0.5."""
    rows, k = x.shape
    blocks = -(-k // BLOCK)
    d = torch.zeros(rows, blocks * BLOCK, dtype=torch.float64, device=x.device)
    d[:, :k] = x
    d = d.view(rows, blocks, BLOCK)
    top = d.abs().max(2, keepdim=True).values
    e = torch.where(top > 0, torch.frexp(top).exponent - 1, torch.full_like(top, -1000, dtype=torch.int32))
    unit = _unit((e - 2).clamp(-127, 125))
    t = d / unit
    step = _unit(torch.frexp(t).exponent.clamp(min=1) - 2)
    r = (torch.round(t / step) * step).clamp(-6.0, 6.0) * unit  # torch.round: halves to even
    return r.view(rows, -1)[:, :k]


def _exact_parts(parts, k):
    codes, scale = parts
    both = torch.stack([codes.bitwise_and(15), codes.bitwise_right_shift(4)], -1).flatten(1).to(torch.int64)
    exp2, frac, neg = (both >> 1) & 3, both & 1, both >> 3
    mag = torch.where(exp2 == 0, 0.5 * frac.double(), (1.0 + 0.5 * frac.double()) * _unit(exp2 - 1))
    unit = _unit(scale.to(torch.int64) - 127)
    return ((1 - 2 * neg) * mag * unit.repeat_interleave(BLOCK, 1))[:, :k]


def exact(case, seed):
    st = prepare(case, seed)
    op, k, x = case["op"], case["k"], st["x"]
    if op == "quantize":
        sides = {"1": [x], "0": [x.t()], "both": [x, x.t()]}[case["axis"]]
        return [_exact_round(s) for s in sides]
    if op == "train":
        w, dy = st["w"], st["dy"]
        return [_exact_round(x) @ _exact_round(w).t(), _exact_round(dy) @ _exact_round(w.t()).t(),
                _exact_round(dy.t()) @ _exact_round(x.t()).t()]
    a = _exact_parts(x, k) if op == "matmul" else _exact_round(x)
    return a @ _exact_parts(st["w"], k).t()
