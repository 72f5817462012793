"""What the MXFP4 operators refuse, checked without a GPU: every refusal comes before any GPU call."""

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def mx():
    from gpumon.ops import mx as m

    return m


@pytest.fixture(scope="module")
def H():
    from gpumon import hip

    return hip()


def test_tensors_on_the_cpu_and_other_types_are_refused(mx):
    x = torch.zeros(4, 32)
    for f in (mx.quantize, mx.quantize_both, lambda t: mx.linear(t, None), lambda t: mx.linear_train(t, t),
              lambda t: mx.linear_grad(t, None)):
        with pytest.raises(ValueError, match="on a GPU"):
            f(x)
        with pytest.raises(TypeError, match="tensor"):
            f([1.0])
    for f in (lambda: mx.matmul(x, x), lambda: mx.dequantize(x)):
        with pytest.raises(TypeError, match="MxTensor"):
            f()
    with pytest.raises(TypeError, match="uint8"):
        mx.MxTensor.pack(x, x, 32)
    u = torch.zeros(4, 16, dtype=torch.uint8)
    with pytest.raises(ValueError, match="on a GPU"):
        mx.MxTensor.pack(u, u, 32)
    for rows, k in ((-1, 5), (3, 0)):
        with pytest.raises(ValueError, match="rows >= 0 and k >= 1"):
            mx.MxTensor(rows, k, "cpu")


def test_products_of_other_sizes_are_refused(mx):
    a, b = mx.MxTensor(3, 64, "cpu"), mx.MxTensor(5, 65, "cpu")
    with pytest.raises(ValueError, match="second sizes differ"):
        mx.matmul(a, b)
    with pytest.raises(TypeError, match="dtype"):
        mx.matmul(a, a, torch.float64)
    with pytest.raises(TypeError, match="dtype"):
        mx.dequantize(a, torch.int32)


def _copies(q):
    import copy
    import io
    import pickle

    file = io.BytesIO()
    torch.save(q, file)
    file.seek(0)
    return copy.deepcopy(q), copy.copy(q), pickle.loads(pickle.dumps(q)), torch.load(file, weights_only=False)


@pytest.mark.parametrize("rows,k", [(1, 1), (3, 64), (17, 1337)])
def test_a_copied_matrix_uses_its_own_memory(mx, rows, k):
    q = mx.MxTensor(rows, k, "cpu")
    q.buf.copy_(torch.arange(q.buf.numel()).to(torch.uint8))
    for c in _copies(q):
        assert c.shape == q.shape and c.device == q.device
        assert c._codes == c.buf.data_ptr() and c._scales - c._codes == q._scales - q._codes
        assert torch.equal(c.codes, q.codes) and torch.equal(c.scales, q.scales)


def test_a_matrix_is_not_rebuilt_from_another_buffer(mx):
    q = mx.MxTensor(17, 1337, "cpu")
    remake, (buf, rows, k) = q.__reduce__()
    for bad in (buf[:-1], buf.view(torch.int8), torch.cat((buf, buf))[::2]):
        with pytest.raises(ValueError, match="buffer"):
            remake(bad, rows, k)


def test_matrices_off_the_gpu_are_refused(mx):
    a, b = mx.MxTensor(3, 64, "cpu"), mx.MxTensor(5, 64, "cpu")
    for f in (lambda: mx.matmul(a, b), lambda: mx.dequantize(a)):
        with pytest.raises(ValueError, match="on a GPU"):
            f()

P = 1 << 20  # an aligned address that nothing here reaches


@pytest.mark.parametrize("over,match", [
    ({"dtype": "f64"}, "dtype"), ({"rows": -1}, "rows"), ({"k": 0}, "k >= 1"), ({"stride": 31}, "stride"),
    ({"rows": 1 << 31}, "limits"), ({"rows": 1 << 20, "k": 1 << 20, "stride": 1 << 20}, "limits"), ({"x": 0}, "null"),
    ({"codes": 0}, "null"), ({"scales": 0}, "null"), ({"x": P + 1}, "aligned"), ({"codes": P + 8}, "aligned"),
    ({"scales": P + 2}, "aligned")])
def test_native_quantize_refuses(H, over, match):
    ok = dict(dev=0, x=P, dtype="bf16", rows=4, k=32, stride=32, by_column=False, codes=P, scales=P)
    with pytest.raises(ValueError, match=match):
        H.mx_quantize(**{**ok, **over})
    both = {**ok, **over}
    both.pop("by_column")
    codes, scales = both.pop("codes"), both.pop("scales")
    with pytest.raises(ValueError, match=match):
        H.mx_quantize_both(row_codes=codes, row_scales=scales, col_codes=codes, col_scales=scales, **both)
    back = {**ok, **over}
    back.pop("by_column")
    with pytest.raises(ValueError, match=match):
        H.mx_dequantize(out=back.pop("x"), **back)


def test_native_quantize_by_column_refuses_no_rows(H):
    with pytest.raises(ValueError, match="rows"):
        H.mx_quantize(0, P, "bf16", 0, 32, 32, True, P, P)


@pytest.mark.parametrize("over,match", [
    ({"dtype": "f64"}, "dtype"), ({"m": -1}, "m and n"), ({"n": -1}, "m and n"), ({"k": 0}, "k >= 1"),
    ({"stride": 47}, "stride"), ({"m": 1 << 31}, "limits"), ({"n": 1 << 20, "k": 1 << 20, "stride": 1 << 20}, "limits"),
    ({"m": 1 << 30, "n": 1 << 30, "stride": 1 << 30}, "limits"), ({"a_codes": 0}, "null"), ({"b_scales": 0}, "null"),
    ({"c": 0}, "null"), ({"a_codes": P + 4}, "aligned"), ({"b_scales": P + 1}, "aligned"), ({"c": P + 1}, "aligned")])
def test_native_product_refuses(H, over, match):
    ok = dict(dev=0, a_codes=P, a_scales=P, b_codes=P, b_scales=P, m=4, n=48, k=64, c=P, dtype="bf16", stride=48)
    with pytest.raises(ValueError, match=match):
        H.mx_product(**{**ok, **over})


def test_native_linear_refuses_a_small_workspace(H):
    need = H.mx_linear_workspace(300, 400, 500, "bf16")
    assert need > 0
    with pytest.raises(ValueError, match="workspace"):
        H.mx_linear(0, P, "bf16", 500, P, P, 300, 400, 500, P, 400, P, need - 1)


def test_native_training_step_refuses(H):
    m, n, k = 40, 50, 60
    saved, ws = H.mx_linear_train_saved(m, n, k), H.mx_linear_train_workspace(m, n, k)
    ok = dict(dev=0, x=P, dtype="bf16", x_stride=k, w=P, w_dtype="f32", w_stride=k, m=m, n=n, k=k, y=P, y_stride=n, saved=P,
              saved_bytes=saved, workspace=P, workspace_bytes=ws)
    for over, match in (({"dtype": "f64"}, "dtype"), ({"w_dtype": "i8"}, "w_dtype"), ({"m": 0}, "m and n"),
                        ({"n": 0}, "m and n"), ({"k": 0}, "k >= 1"), ({"x_stride": k - 1}, "stride"),
                        ({"w_stride": k - 1}, "stride"), ({"y_stride": n - 1}, "stride"), ({"x": 0}, "null"),
                        ({"w": 0}, "null"), ({"y": 0}, "null"), ({"saved": 0}, "sizes"), ({"saved_bytes": saved - 1}, "sizes"),
                        ({"workspace_bytes": ws - 1}, "sizes"), ({"workspace": P + 8}, "sizes"), ({"w": P + 2}, "aligned"),
                        ({"x": P + 1}, "aligned"), ({"m": 1 << 28}, "limits")):
        with pytest.raises(ValueError, match=match):
            H.mx_linear_train(**{**ok, **over})
    need = H.mx_linear_grad_workspace(m, n, k)
    ok = dict(dev=0, dy=P, dtype="bf16", dy_stride=n, saved=P, m=m, n=n, k=k, dx=P, dx_stride=k, dw=P, w_dtype="f32",
              dw_stride=k, workspace=P, workspace_bytes=need)
    for over, match in (({"dtype": "f64"}, "dtype"), ({"w_dtype": "i8"}, "w_dtype"), ({"m": 0}, "m and n"),
                        ({"dy_stride": n - 1}, "stride"), ({"dx_stride": k - 1}, "stride"), ({"dw_stride": k - 1}, "stride"),
                        ({"dy": 0}, "null"), ({"saved": 0}, "sizes"), ({"saved": P + 4}, "sizes"),
                        ({"workspace_bytes": need - 1}, "sizes"), ({"dx": P + 1}, "aligned"), ({"dw": P + 2}, "aligned")):
        with pytest.raises(ValueError, match=match):
            H.mx_linear_grad(**{**ok, **over})
