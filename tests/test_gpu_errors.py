"""An error of one call is that call's alone, on a real MI355X: what comes after it on the thread runs."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _too_large():
    from gpumon.ops.load import SyntheticLoad

    load = SyntheticLoad(0, "hbm", hbm_bytes=1 << 44)  # more than any card has
    try:
        load.start()
    finally:
        load.stop()


def _no_such_device():
    from gpumon import hip

    p = torch.zeros(64, 64, device="cuda").data_ptr()
    hip().mx_quantize(torch.cuda.device_count() + 3, p, "f32", 4, 32, 32, False, p, p)


@pytest.mark.parametrize("fail", [_too_large, _no_such_device])
@pytest.mark.parametrize("after", ["torch", "mx", "load"])
def test_what_follows_an_error_runs(fail, after):
    from gpumon.ops import mx
    from gpumon.ops.load import SyntheticLoad

    x = torch.ones(4, 64, device="cuda")
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError):
        fail()
    if after == "torch":
        assert float((x + 1).sum()) == 512
    elif after == "mx":
        assert torch.equal(mx.dequantize(mx.quantize(x)), x)
    else:
        with SyntheticLoad(0, "mfma", mfma_iters=256):
            pass
