"""Quantised matrices (gpumon.ops.mx.MxTensor) off the GPU."""

import pytest

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("k", [1, 70, 1337])
def test_parts_of_a_matrix_without_rows(k):
    from gpumon.ops import mx

    codes, scales = mx.MxTensor(0, k, "cpu").parts()
    blocks = -(-k // 32)
    assert codes.shape == (0, blocks * 16) and scales.shape == (0, blocks)
    assert codes.dtype == scales.dtype == torch.uint8
