"""Every product kernel of the MXFP4 operators, by name: which sizes take it (CPU), and its results (MI355X).

Operands are whole numbers of the 4-bit grid (0, 1, 2, 3, 4, 6 and their negatives), which every scale
of a block of them holds exactly. Their products' sums stay below 2^24 for k up to 2^24 / 36 = 466033, so
they are exact in 32 bits in any order, and a result is the exact sum rounded once: equality, at any
length. An element left out, counted twice or rounded on the way shows.
"""

import pytest

torch = pytest.importorskip("torch")

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAMES = {BF16: "bf16", F16: "f16", F32: "f32"}

# m, n, k off the tiles, the quads (128) and the groups (512), but for a few of them
PRODUCTS = {
    "256x256": [(1987, 8081, 523), (3905, 8111, 1025), (4096, 4096, 4096)],  # the second: two rounds of tiles
    "256x128": [(2047, 4001, 4200), (8681, 3798, 65)],  # the second: four rounds
    "128x128": [(2047, 3001, 1333), (4099, 4301, 700)],
    "64x128": [(2047, 3001, 300), (1030, 4100, 8300)],
    "64x64": [(1500, 1400, 700), (67, 70, 65), (2100, 1100, 4100)],
    "64x64/2": [(916, 337, 10650), (167, 2511, 13482)],
    "64x64/3": [(679, 322, 8005), (924, 253, 8476)],
    "64x64/4": [(115, 73, 3748), (85, 369, 5384)],
    "64x64/5": [(112, 56, 4611), (177, 33, 6219)],
    "64x64/6": [(70, 66, 9000), (106, 100, 5765)],
    "64x64/7": [(300, 20, 12345), (158, 294, 9860)],
    "64x64/8": [(224, 65, 11657), (130, 200, 100000)],
    "few16": [(1, 1, 100000), (1, 300, 4097), (5, 3, 33333), (16, 70, 2500), (13, 50, 700)],
    "few32": [(17, 300, 9999), (32, 4096, 513)],
    "few32x2": [(31, 4100, 4700), (20, 5000, 100)],
    "few64": [(40, 100, 100000), (64, 4000, 1100), (33, 65, 300)],
    "few64x2": [(50, 4100, 5005), (64, 4200, 2000)],
}
LINEARS = {
    "way1": [(1, 300, 30001), (1, 5000, 700)],
    "way4": [(2, 300, 12345), (4, 4700, 1300), (3, 33, 65)],
    "way8": [(5, 300, 12001), (8, 4000, 1000)],
    "way8x2": [(7, 4200, 5003), (8, 5000, 300)],
    "few16": [(9, 300, 2100), (8, 300, 50001)],
    "few32": [(20, 300, 2100)],
    "64x64": [(700, 800, 300)],
}
FLAT = [(name, s) for name, sizes in PRODUCTS.items() for s in sizes]
FLAT_LINEAR = [(name, s) for name, sizes in LINEARS.items() for s in sizes]


@pytest.fixture(scope="module")
def H():
    from gpumon import hip

    return hip()


@pytest.mark.parametrize("name,size", FLAT, ids=lambda v: v if isinstance(v, str) else "x".join(map(str, v)))
def test_product_sizes_take_the_kernel_they_stand_for(H, name, size):
    assert H.mx_product_kernel(*size) == name


@pytest.mark.parametrize("name,size", FLAT_LINEAR, ids=lambda v: v if isinstance(v, str) else "x".join(map(str, v)))
def test_linear_sizes_take_the_kernel_they_stand_for(H, name, size):
    for dtype in ("bf16", "f16", "f32"):
        assert H.mx_linear_kernel(*size, dtype) == name


def test_no_kernel_is_without_a_size(H):
    """Sizes over the whole range take no kernel that the tables above do not hold."""
    import math
    import random

    r = random.Random(1)
    for _ in range(20000):
        m, n, k = (round(math.exp(r.uniform(0, math.log(20000)))) for _ in range(3))
        assert H.mx_product_kernel(m, n, k) in PRODUCTS, (m, n, k)
        name = H.mx_linear_kernel(m, n, k, r.choice(["bf16", "f16", "f32"]))
        assert name in PRODUCTS or name in LINEARS, (m, n, k)


TRAININGS = {  # the tile of both gradients' launch, "" for a launch each
    "64x64": [(631, 62, 2101)], "64x128": [(75, 73, 7890), (40, 520, 9000)], "128x128": [(1098, 65, 8181)],
    "256x128": [(3534, 129, 8504)], "256x256": [(1166, 1203, 6308)], "": [(2449, 8475, 6300)],
}


def test_training_sizes_take_the_kernel_they_stand_for(H):
    for name, sizes in TRAININGS.items():
        for size in sizes:
            assert H.mx_linear_grad_kernel(*size) == name, size


def whole(rows, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    grid = torch.tensor([0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6.0], device="cuda")
    return grid[torch.randint(0, 11, (rows, k), generator=g, device="cuda")]


@pytest.mark.gpu
@pytest.mark.parametrize("name,size", FLAT, ids=lambda v: v if isinstance(v, str) else "x".join(map(str, v)))
def test_products_of_whole_numbers(name, size):
    from gpumon.ops import mx

    m, n, k = size
    a, b = whole(m, k, m + k), whole(n, k, n)
    want = a @ b.t()
    qa, qb = mx.quantize(a), mx.quantize(b)
    for dtype in NAMES:
        assert torch.equal(mx.matmul(qa, qb, dtype), want.to(dtype)), (name, size, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("name,size", FLAT_LINEAR, ids=lambda v: v if isinstance(v, str) else "x".join(map(str, v)))
def test_linear_layers_of_whole_numbers(name, size):
    from gpumon.ops import mx

    m, n, k = size
    x, w = whole(m, k, m + k), whole(n, k, n)
    want = x @ w.t()
    q = mx.quantize(w)
    for dtype in NAMES:
        assert torch.equal(mx.linear(x.to(dtype), q), want.to(dtype)), (name, size, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [s for sizes in TRAININGS.values() for s in sizes])
@pytest.mark.parametrize("dtype,w_dtype", [(BF16, BF16), (F16, F16), (F32, F32), (F16, F32)])
def test_training_steps_of_whole_numbers(m, n, k, dtype, w_dtype):
    """Gradients in one launch by tiles of every size, and each in its own (other types, and the last size)."""
    from gpumon.ops import mx

    x, w, dy = whole(m, k, 1), whole(n, k, 2), whole(m, n, 3)
    y, saved = mx.linear_train(x.to(dtype), w.to(w_dtype))
    dx, dw = mx.linear_grad(dy.to(dtype), saved)
    assert torch.equal(y, (x @ w.t()).to(dtype))
    assert torch.equal(dx, (dy @ w).to(dtype))
    assert torch.equal(dw, (dy.t() @ x).to(w_dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("name", [n for n in PRODUCTS])
def test_results_with_gaps_between_their_rows(H, name):
    """Native entry: rows on and off 64 bytes apart, the gaps and the rows around them left as they were."""
    from gpumon.ops import mx

    s = torch.cuda.current_stream().cuda_stream
    m, n, k = PRODUCTS[name][0]
    a, b = whole(m, k, 1), whole(n, k, 2)
    want = a @ b.t()
    qa, qb = mx.quantize(a), mx.quantize(b)
    need = H.mx_product_workspace(m, n, k)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    for dtype in NAMES:
        for stride, first in ((n + 13, 3), ((n + 127) // 64 * 64, 0)):
            out = torch.full((m + 2, stride), 5.0, dtype=dtype, device="cuda")
            H.mx_product(0, qa.codes.data_ptr(), qa.scales.data_ptr(), qb.codes.data_ptr(), qb.scales.data_ptr(), m, n, k,
                         out[1:, first:].data_ptr(), NAMES[dtype], stride, ws.data_ptr(), need, s)
            inner = out[1:m + 1, first:first + n]
            assert torch.equal(inner, want.to(dtype)), (name, dtype, stride)
            inner.fill_(5.0)
            assert (out == 5.0).all(), (name, dtype, stride)
