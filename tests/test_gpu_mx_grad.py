"""gpumon.ops.mx.linear_grad: each gradient by itself and both together, on a real MI355X."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("m,n,k", [(631, 62, 2101), (40, 1500, 9000), (1700, 40, 3000), (9000, 70, 80), (20, 3000, 500), (300, 20, 12345),
                                   (70, 5000, 200), (75, 73, 7890), (1166, 1203, 6308), (2449, 8475, 6300)])
@pytest.mark.parametrize("dtype,w_dtype", [(F32, F32), (BF16, BF16), (BF16, F32)])
def test_a_gradient_does_not_depend_on_what_else_is_asked_for(m, n, k, dtype, w_dtype):
    """Bit for bit, also where one alone would have its k in parts or take the kernel for few rows. Values
    over so many powers of two that sums round at nearly every addition."""
    from gpumon.ops import mx

    g = torch.Generator(device="cuda").manual_seed(m + k)

    def wide(r, c):  # a power of two for every 32 rows and every 32 columns
        by = [torch.exp2(torch.randint(-10, 11, (-(-v // 32),), generator=g, device="cuda").float()).repeat_interleave(32)[:v]
              for v in (r, c)]
        return torch.randn(r, c, generator=g, device="cuda") * by[0][:, None] * by[1]

    x, w, dy = wide(m, k), wide(n, k), wide(m, n)
    _, saved = mx.linear_train(x.to(dtype), w.to(w_dtype))
    dy = dy.to(dtype)
    dx, dw = mx.linear_grad(dy, saved)
    assert torch.equal(mx.linear_grad(dy, saved, need_dw=False)[0], dx)
    assert torch.equal(mx.linear_grad(dy, saved, need_dx=False)[1], dw)
