"""gpumon.ops.mx.quantize over every 16-bit value under every scale, on a real MI355X."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_mx import assert_quantized  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_value_under_every_scale(dtype):
    """Each power of two of the type as a block's maximum, and each value up to it in blocks of that maximum,
    along the rows and down the columns."""
    from gpumon.ops import mx

    v = torch.arange(65536).to(torch.int32).to(torch.int16).view(dtype)
    v = v[torch.isfinite(v)].double()
    info = torch.finfo(dtype)
    low = round(torch.log2(torch.tensor(info.smallest_normal * info.eps, dtype=torch.float64)).item())
    high = int(torch.log2(torch.tensor(info.max, dtype=torch.float64)).item())
    blocks = []
    for e in range(low, high + 1):
        some = v[v.abs() <= 2.0 ** e]
        some = torch.cat([some, some.new_zeros(-len(some) % 31)]).view(-1, 31)
        blocks.append(torch.cat([some, torch.full((len(some), 1), 2.0 ** e, dtype=torch.float64)], 1))
    x = torch.cat(blocks).to(dtype)
    scales = mx.quantize(x.cuda()).parts()[1].unique().tolist()
    assert scales == list(range(max(low + 125, 0), high + 126))
    assert_quantized(mx.quantize(x.cuda()), x)
    assert_quantized(mx.quantize(x.t().contiguous().cuda(), 0), x)


def test_two_matrices_whose_tiles_are_too_many_for_one_launch():
    """A training step's x and w together have 2^23 tiles; each for itself is within the limit."""
    from gpumon.ops import mx

    m, n, k = (1 << 28) - 200, 16, 1
    grid = torch.tensor([0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6.0], device="cuda").bfloat16()
    x = grid[torch.randint(0, 11, (m, k), device="cuda")]
    w = grid[torch.randint(0, 11, (n, k), device="cuda")]
    y, saved = mx.linear_train(x, w)
    for at in (0, m // 2, m - (1 << 20)):
        rows = slice(at, at + (1 << 20))
        assert torch.equal(y[rows], x[rows] * w.t())
    del y
    dy = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    dy[-100:] = grid[torch.randint(0, 11, (100, n), device="cuda")]
    dx, dw = mx.linear_grad(dy, saved)
    assert torch.equal(dx[-100:], (dy[-100:].float() @ w.float()).bfloat16()) and not dx[:-100].any()
    assert torch.equal(dw, (dy[-100:].float().t() @ x[-100:].float()).bfloat16())
