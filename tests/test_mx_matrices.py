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


P = 1 << 20  # an aligned address that nothing here reaches


def test_more_tiles_than_a_launch_takes_are_refused():
    """A launch has fewer than 2^32 threads: 2^23 tiles of 32 rows x 512 columns are one too many."""
    from gpumon import hip

    H, rows = hip(), (1 << 28) - 16
    with pytest.raises(ValueError, match="limits"):
        H.mx_quantize(0, P, "bf16", rows, 1, 1, True, P, P)
    with pytest.raises(ValueError, match="limits"):
        H.mx_quantize_both(0, P, "bf16", rows, 1, 1, P, P, P, P)
    m, n, k = rows, 16, 1
    sizes = H.mx_linear_train_saved(m, n, k), H.mx_linear_train_workspace(m, n, k)
    with pytest.raises(ValueError, match="limits"):
        H.mx_linear_train(0, P, "bf16", k, P, "bf16", k, m, n, k, P, n, P, sizes[0], P, sizes[1])
