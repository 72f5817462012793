"""gpumon.ops.mx and torch's gradients: refused where they would be lost, usable where they are taken care of."""

import pytest

torch = pytest.importorskip("torch")


def test_what_counts_as_an_input_with_a_gradient():
    from torch.autograd import forward_ad

    from gpumon.ops import mx

    plain, leaf = torch.ones(2, 32), torch.ones(2, 32, requires_grad=True)
    mx._check_constant(plain, "x")
    for t in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="requires a gradient"):
            mx._check_constant(t, "x")
        mx._check_constant(t.detach(), "x")
        with torch.no_grad():
            mx._check_constant(t, "x")
        with torch.inference_mode():
            mx._check_constant(t, "x")
    with forward_ad.dual_level():
        mx._check_constant(plain, "x")
        with pytest.raises(ValueError, match="tangent"):
            mx._check_constant(forward_ad.make_dual(plain, plain), "x")


@pytest.mark.gpu
def test_linear_layers_refuse_inputs_whose_gradient_they_would_lose():
    from torch.autograd import forward_ad

    from gpumon.ops import mx

    x, w, dy = (torch.randn(s, device="cuda") for s in ((5, 70), (9, 70), (5, 9)))
    xg, wg, dg = (t.clone().requires_grad_() for t in (x, w, dy))
    q = mx.quantize(wg)  # no tensor, so nothing that could be differentiated
    _, saved = mx.linear_train(x, w)
    calls = [lambda: mx.linear(xg, q), lambda: mx.linear(xg * 1, q), lambda: mx.linear_train(xg, w),
             lambda: mx.linear_train(x, wg), lambda: mx.linear_grad(dg, saved)]
    for call in calls:
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
        with torch.no_grad():
            call()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        for call in (lambda: mx.linear(dual, q), lambda: mx.linear_train(dual, w)):
            with pytest.raises(ValueError, match="tangent"):
                call()


@pytest.mark.gpu
def test_the_layer_as_a_function_of_torch():
    from gpumon.ops import mx

    class Linear(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            y, ctx.layer = mx.linear_train(x, w)
            return y

        @staticmethod
        def backward(ctx, dy):
            return mx.linear_grad(dy, ctx.layer, *ctx.needs_input_grad)

    g = torch.Generator(device="cuda").manual_seed(1)
    x, w, t = (torch.randn(s, generator=g, device="cuda") for s in ((4, 10, 70), (9, 70), (4, 10, 9)))
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = Linear.apply(torch.tanh(xg), wg)
    (y * t).sum().backward()
    want, saved = mx.linear_train(torch.tanh(x), w)
    dx, dw = mx.linear_grad(t, saved)
    assert torch.equal(y, want) and torch.equal(wg.grad, dw)
    assert torch.equal(xg.grad, torch.autograd.grad(torch.tanh(xg), xg, dx)[0])
