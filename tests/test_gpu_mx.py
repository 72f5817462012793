"""MXFP4 operators (gpumon.ops.mx) on a real MI355X against the format's definition in 64 bits.

Codes and scales are determined by the definition (dividing by a power of two is exact), so
quantisation is compared bit for bit. A product's tolerance counts its roundings: every product of
two elements is exact in 32 bits; adding k of them in any order errs by at most
k * 2^-23 * sum |a_i b_i| (each addition by at most one step of 2^-23, in case it truncates), and
the result is rounded once to the output type (half a step, eps / 2 of the value, or half the
smallest subnormal).
"""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF16, F16, F32]
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}  # half the smallest subnormal


@pytest.fixture(scope="module")
def mx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from gpumon.ops import mx as m

    return m


def pow2(e):
    return (e.long() + 1023).bitwise_left_shift(52).view(torch.float64)


def ref_quantize(x):
    """Nibbles [rows, blocks * 32] (zeros past k) and scale bytes [rows, blocks], from the definition, on the CPU."""
    rows, k = x.shape
    blocks = -(-k // 32)
    d = torch.zeros(rows, blocks * 32, dtype=torch.float64)
    d[:, :k] = x.cpu().double()
    b = d.view(rows, blocks, 32)
    bad = ~torch.isfinite(b).all(2)
    amax = b.abs().amax(2).masked_fill(bad, 0)
    e = (torch.frexp(amax)[1].long() - 3).clamp(-127, 125).masked_fill(amax == 0, -127)
    t = b.abs() / pow2(e).unsqueeze(2)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    mid = (grid[1:] + grid[:-1]) / 2
    code = torch.bucketize(t, mid)  # a halfway point goes to the lower neighbour here
    up = (t == mid[code.clamp(max=6)]) & (code % 2 == 1)  # the lower neighbour is odd: to the upper one
    code = code + up.long() + 8 * torch.signbit(b).long()
    code = code.masked_fill(bad.unsqueeze(2), 0)
    return code.view(rows, -1), (e + 127).masked_fill(bad, 255)


def ref_values(code, scale, k):
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    v = torch.where(code >= 8, -grid[code % 8], grid[code % 8]).view(code.shape[0], -1, 32) * pow2(scale - 127).unsqueeze(2)
    v[scale == 255] = float("nan")
    return v.view(code.shape[0], -1)[:, :k]


def ref_round(x):
    return ref_values(*ref_quantize(x), x.shape[1])


def mx_parts(q):
    codes, scales = (t.cpu().long() for t in q.parts())
    return torch.stack([codes & 15, codes >> 4], 2).view(q.rows, -1), scales


def assert_quantized(q, x):
    """q is exactly what the definition makes of x, and zeros in what fills it up."""
    code, scale = ref_quantize(x)
    got, gs = mx_parts(q)
    assert q.shape == tuple(x.shape)
    assert torch.equal(gs, scale)
    assert torch.equal(got, code)
    # nothing but zeros fills it up: as much as the row-major parts laid out anew
    again = type(q).pack(*q.parts(), q.k)
    assert torch.equal(q.codes, again.codes) and torch.equal(q.scales, again.scales)


def assert_product(c, a, b):
    """c against a @ b.T of 64-bit values a, b (NaN rows included), within the product's roundings."""
    dt = c.dtype
    ref = a @ b.t()
    bound = a.shape[1] * 2.0 ** -23 * (a.abs() @ b.abs().t())
    bound = bound * (1 + torch.finfo(dt).eps) + ref.abs() * (torch.finfo(dt).eps / 2) + TINY[dt]
    got = c.cpu().double()
    assert got.shape == ref.shape
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan)
    big = torch.finfo(dt).max
    inf = (ref.abs() > big) & ~nan  # beyond the type: an infinity, or its largest number within the bound
    ok = ((got - ref).abs() <= bound) | nan | (inf & (got.sign() == ref.sign()) & (got.abs() >= big * (1 - 2.0 ** -6)))
    assert ok.all(), (float(((got - ref).abs() - bound).nan_to_num(-1).max()), int((~ok).sum()))


def values(rows, k, dtype, seed=0, special=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g, dtype=torch.float64)
    x *= torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g).double())
    x *= torch.exp2(torch.randint(-3, 4, (1, k), generator=g).double())
    x = x.to(dtype)
    if special and x.numel():
        big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
        flat = x.view(-1)
        flat[::37] = 0
        for j, v in enumerate((-0.0, float("nan"), float("inf"), -float("inf"), big, -big, tiny, tiny / 2, -tiny / 4)):
            flat[(j * 131 + 5) % flat.numel()] = v
    return x.cuda()


SHAPES = [(1, 1), (1, 31), (3, 32), (5, 33), (2, 127), (16, 128), (17, 129), (64, 256), (33, 1000), (128, 130),
          (1, 8192), (257, 511), (1000, 7)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", SHAPES)
def test_quantize_both_directions_bit_for_bit(mx, rows, k, dtype):
    for special in (False, True):
        x = values(rows, k, dtype, rows * 1000 + k, special)
        assert_quantized(mx.quantize(x), x)
        assert_quantized(mx.quantize(x, axis=0), x.t())
        along, down = mx.quantize_both(x)
        assert_quantized(along, x)
        assert_quantized(down, x.t())


def test_every_16_bit_value_at_every_distance_to_the_block_maximum(mx):
    """Each finite bf16 and f16 value, next to maxima 1 to 2^7 times as large (so every rounding border
    and both sides of it come up), as a block of its own."""
    for dtype in (BF16, F16):
        v = torch.arange(65536).to(torch.int32).to(torch.int16).view(dtype)
        v = v[torch.isfinite(v)]
        for shift in range(8):
            top = v.double().abs() * 2.0 ** shift * 1.25
            top = torch.minimum(top, torch.tensor(float(torch.finfo(dtype).max), dtype=torch.float64)).to(dtype)
            x = torch.zeros(len(v), 32, dtype=dtype)
            x[:, 3], x[:, 30] = v, top
            assert_quantized(mx.quantize(x.cuda()), x)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strides_and_views(mx, dtype):
    base = values(70, 400, dtype, 5)
    for x in (base[3:60, 7:390], base[::2], base.t(), base.t()[5:333], base[:, 5:6], base[4:5], base[:1].expand(9, 400),
              base[:, :1].expand(70, 50), base[:, ::3]):
        assert_quantized(mx.quantize(x), x)
        assert_quantized(mx.quantize(x, 0), x.t())
        along, down = mx.quantize_both(x)
        assert_quantized(along, x)
        assert_quantized(down, x.t())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 40), (17, 129), (65, 1000)])
def test_dequantize_and_parts(mx, rows, k, dtype):
    x = values(rows, k, F32, 11, True)
    q = mx.quantize(x)
    want = ref_round(x).to(F32).to(dtype)
    got = mx.dequantize(q, dtype).cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7), want.nan_to_num(7))
    p = mx.MxTensor.pack(*q.parts(), k)
    assert torch.equal(p.buf, q.buf)


def test_every_code_under_every_scale_dequantizes_exactly(mx):
    codes = torch.arange(16, dtype=torch.uint8)
    codes = (codes | (codes.flip(0) << 4)).repeat(256, 1).cuda()
    scales = torch.arange(256).view(256, 1).to(torch.uint8).cuda()
    q = mx.MxTensor.pack(codes, scales, 32)
    code, scale = mx_parts(q)
    ref = ref_values(code, scale, 32)
    for dtype in TYPES:
        got = mx.dequantize(q, dtype).cpu()
        want = ref.to(F32).to(dtype)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7), want.nan_to_num(7))


def test_pack_ignores_what_is_past_k(mx):
    x = values(5, 64, F32, 1)
    codes, scales = mx.quantize(x).parts()
    for k in (63, 61, 50, 33):
        q = mx.MxTensor.pack(codes, scales, k)
        assert torch.equal(mx.dequantize(q), mx.dequantize(mx.MxTensor.pack(codes, scales, 64))[:, :k])
        y = mx.matmul(q, q, F32)
        v = mx.dequantize(q).cpu().double()
        assert_product(y, v, v)


PRODUCTS = [(1, 1, 1), (1, 16, 32), (1, 1000, 4096), (2, 33, 64), (7, 130, 129), (15, 64, 1000), (16, 256, 512),
            (17, 48, 640), (31, 1411, 256), (33, 65, 300), (64, 64, 128), (65, 257, 1025), (100, 100, 100),
            (128, 128, 256), (129, 300, 384), (200, 1000, 2500), (256, 256, 256), (257, 511, 768), (300, 260, 130),
            (512, 512, 1152), (513, 1030, 2048), (777, 1411, 2999), (1024, 2048, 640), (2100, 1100, 300), (1, 70000, 96),
            (5000, 3, 200), (3, 5, 100000), (40, 40, 20000), (70, 66, 9000), (130, 200, 8192), (500, 300, 33000), (300, 20, 12345), (2000, 2100, 300), (3600, 1029, 1300)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul_within_its_roundings(mx, m, n, k):
    for i, dtype in enumerate(TYPES):
        a, b = values(m, k, F32, m + k + i), values(n, k, BF16, n + i)
        assert_product(mx.matmul(mx.quantize(a), mx.quantize(b), dtype), ref_round(a), ref_round(b))


def test_matmul_of_whole_numbers_is_exact(mx):
    """Elements 0..6 with one scale: sums of whole numbers below 2^24 are exact in any order, so each
    element is where it belongs and nothing is counted twice."""
    g = torch.Generator().manual_seed(2)
    for m, n, k in ((300, 500, 700), (1, 8192, 4096), (16, 1000, 3000), (48, 333, 2222), (1100, 1300, 520), (2048, 2048, 2048)):
        pick = torch.tensor([0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6.0])
        a, b = pick[torch.randint(0, 11, (m, k), generator=g)], pick[torch.randint(0, 11, (n, k), generator=g)]
        a[:, ::32], b[:, ::32] = 6, -6  # every block has the same scale
        c = mx.matmul(mx.quantize(a.cuda()), mx.quantize(b.cuda()), F32)
        assert torch.equal(c, a.cuda() @ b.cuda().t())


@pytest.mark.parametrize("m,n,k", [(1, 100, 500), (20, 300, 500), (300, 500, 700), (520, 600, 260)])
def test_scales_of_every_size_and_nan_blocks(mx, m, n, k):
    """Scale bytes over the whole range, some of them NaN:
    a NaN block makes its row or column NaN, codes of zero or not, and nothing else."""
    g = torch.Generator().manual_seed(m)
    blocks = -(-k // 32)

    def operand(rows, lo, hi, seed):
        codes = torch.randint(0, 256, (rows, blocks * 16), generator=g).to(torch.uint8)
        scales = torch.randint(lo, hi, (rows, blocks), generator=g)
        if rows > 3:
            scales[rows // 2, blocks - 1] = 255
            scales[3, 0] = 255
            codes[3] = 0
        q = mx.MxTensor.pack(codes.cuda(), scales.to(torch.uint8).cuda(), k)
        return q, ref_values(*mx_parts(q), k)

    for lo, hi in ((0, 100), (100, 155), (150, 255)):
        (a, av), (b, bv) = operand(m, lo, hi, 1), operand(n, 254 - hi + 1, 255 - lo, 2)
        for dtype in (BF16, F32):
            assert_product(mx.matmul(a, b, dtype), av, bv)


def test_layouts_of_results_leave_their_surroundings_alone(mx):
    """Native entry: a result whose rows lie apart, the gaps and what follows left as they were."""
    from gpumon import hip

    H = hip()
    s = torch.cuda.current_stream().cuda_stream
    for m, n, k, dt in ((5, 33, 70, BF16), (130, 257, 300, F16), (300, 301, 129, F32), (1, 50, 1000, BF16)):
        a, b = values(m, k, F32, 1), values(n, k, F32, 2)
        qa, qb = mx.quantize(a), mx.quantize(b)
        out = torch.full((m + 2, n + 13), 5.0, dtype=dt, device="cuda")
        need = H.mx_product_workspace(m, n, k)
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        H.mx_product(0, qa.codes.data_ptr(), qa.scales.data_ptr(), qb.codes.data_ptr(), qb.scales.data_ptr(), m, n, k,
                     out[1:, 3:].data_ptr(), mx.DTYPES[dt], n + 13, ws.data_ptr(), need, s)
        assert_product(out[1:m + 1, 3:n + 3], ref_round(a), ref_round(b))
        rest = out.clone()
        rest[1:m + 1, 3:n + 3] = 5.0
        assert (rest == 5.0).all()
        back = torch.full((m + 2, k + 5), 5.0, dtype=dt, device="cuda")
        H.mx_dequantize(0, qa.codes.data_ptr(), qa.scales.data_ptr(), m, k, back[1:, 2:].data_ptr(), mx.DTYPES[dt], k + 5, s)
        assert torch.equal(back[1:m + 1, 2:k + 2], mx.dequantize(qa, dt))
        rest = back.clone()
        rest[1:m + 1, 2:k + 2] = 5.0
        assert (rest == 5.0).all()


LINEARS = [(1, 1, 1), (1, 17, 31), (1, 1000, 1000), (1, 8192, 1024), (2, 100, 4096), (5, 7001, 333), (13, 500, 5005),
           (16, 64, 256), (17, 300, 129), (31, 33, 2000), (32, 512, 512), (33, 200, 700), (64, 1000, 1024), (65, 100, 100),
           (128, 300, 2050), (300, 600, 520), (1000, 130, 260)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", LINEARS)
def test_linear_within_its_roundings(mx, m, n, k, dtype):
    x, w = values(m, k, dtype, m + n, False), values(n, k, BF16, k)
    assert_product(mx.linear(x, mx.quantize(w)), ref_round(x), ref_round(w))


@pytest.mark.parametrize("m", [1, 3, 16, 40, 200])
def test_linear_with_nan_rows_strides_and_leading_dimensions(mx, m):
    k, n = 600, 200
    w = values(n, k, BF16, 3)
    wq, wv = mx.quantize(w), ref_round(w)
    x = values(m, k, BF16, 4, True)
    assert_product(mx.linear(x, wq), ref_round(x), wv)
    wide = values(m, k + 9, F16, 5)
    assert_product(mx.linear(wide[:, 4:k + 4], wq), ref_round(wide[:, 4:k + 4]), wv)
    x3 = values(2 * m, k, BF16, 6).view(2, m, k)
    y = mx.linear(x3, wq)
    assert y.shape == (2, m, n)
    assert_product(y.view(-1, n), ref_round(x3.view(-1, k)), wv)
    assert_product(mx.linear(x3.transpose(0, 1), wq).reshape(-1, n), ref_round(x3.transpose(0, 1).reshape(-1, k)), wv)
    assert_product(mx.linear(x3[0, 0], wq).view(1, n), ref_round(x3[0, :1]), wv)
    assert mx.linear(x[:0], wq).shape == (0, n)


@pytest.mark.parametrize("dtype,w_dtype", [(BF16, BF16), (F16, F32), (F32, BF16)])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (5, 33, 70), (130, 64, 100), (300, 257, 131), (613, 1000, 337), (40, 520, 9000),
                                   (9000, 70, 80), (1200, 1300, 2100)])
def test_training_step_against_the_formulas(mx, m, n, k, dtype, w_dtype):
    x, w, dy = values(m, k, dtype, 1), values(n, k, w_dtype, 2), values(m, n, dtype, 3)
    y, saved = mx.linear_train(x, w)
    dx, dw = mx.linear_grad(dy, saved)
    assert (y.dtype, dx.dtype, dw.dtype) == (dtype, dtype, w_dtype)
    assert_product(y, ref_round(x), ref_round(w))
    assert_product(dx, ref_round(dy), ref_round(w.t()))
    assert_product(dw, ref_round(dy.t()), ref_round(x.t()))
    only_dx, none = mx.linear_grad(dy, saved, need_dw=False)
    assert none is None and torch.equal(only_dx, dx)
    none, only_dw = mx.linear_grad(dy, saved, need_dx=False)
    assert none is None and torch.equal(only_dw, dw)


def test_training_step_against_differences(mx):
    """Where quantising is the identity (whole numbers up to 6 in blocks whose maximum is 6, both ways)
    the layer is linear, so its gradients are exactly the differences of its outputs."""
    m, n, k = 64, 32, 96
    g = torch.Generator().manual_seed(9)

    def grid(r, c):
        v = torch.tensor([0, 1, 2, 3, 4, -1, -2, -3, -4.0])[torch.randint(0, 9, (r, c), generator=g)]
        i = torch.arange(r).view(-1, 1)
        v[(i + torch.arange(c)) % 32 == 0] = 6  # one in every block of either direction
        return v.cuda()

    x, w, dy = grid(m, k), grid(n, k), grid(m, n)
    y, saved = mx.linear_train(x, w)
    dx, dw = mx.linear_grad(dy, saved)

    def loss(x, w):
        return float((mx.linear_train(x, w)[0].double() * dy.double()).sum())

    base = loss(x, w)
    for i, j in ((0, 1), (5, 90), (63, 95), (31, 33)):
        if x[i, j] == 6:
            continue
        x2 = x.clone()
        x2[i, j] = 3.0 if x[i, j] == 2 else 2.0
        assert loss(x2, w) - base == float(dx[i, j]) * float(x2[i, j] - x[i, j])
    for i, j in ((0, 1), (5, 90), (31, 95), (30, 33)):
        if w[i, j] == 6:
            continue
        w2 = w.clone()
        w2[i, j] = 3.0 if w[i, j] == 2 else 2.0
        assert loss(x, w2) - base == float(dw[i, j]) * float(w2[i, j] - w[i, j])


def test_training_step_without_rows(mx):
    w = values(40, 50, BF16, 1)
    y, saved = mx.linear_train(torch.empty(0, 50, dtype=BF16, device="cuda"), w)
    dx, dw = mx.linear_grad(torch.empty(0, 40, dtype=BF16, device="cuda"), saved)
    assert y.shape == (0, 40) and dx.shape == (0, 50) and dw.shape == (40, 50) and not dw.any()


def test_two_layers_trained_and_served_together(mx):
    """A run as it is used: two layers' training steps in a row, a weight update, the new weights
    quantised and served, one token and a prompt."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(96, 160, generator=g).to(BF16).cuda()
    w1 = (torch.randn(200, 160, generator=g) / 12).to(BF16).cuda()
    w2 = (torch.randn(72, 200, generator=g) / 14).to(BF16).cuda()
    t = torch.randn(96, 72, generator=g).to(BF16).cuda()
    h, s1 = mx.linear_train(x, w1)
    act = torch.relu(h)
    y, s2 = mx.linear_train(act, w2)
    dy = (y.float() - t.float()).to(BF16)
    dact, dw2 = mx.linear_grad(dy, s2)
    dh = dact * (h > 0)
    dx, dw1 = mx.linear_grad(dh, s1)
    assert_product(h, ref_round(x), ref_round(w1))
    assert_product(y, ref_round(act), ref_round(w2))
    assert_product(dact, ref_round(dy), ref_round(w2.t()))
    assert_product(dw2, ref_round(dy.t()), ref_round(act.t()))
    assert_product(dx, ref_round(dh), ref_round(w1.t()))
    assert_product(dw1, ref_round(dh.t()), ref_round(x.t()))
    n1, n2 = w1 - 0.01 * dw1, w2 - 0.01 * dw2
    q1, q2 = mx.quantize(n1), mx.quantize(n2)
    for rows in (x[:1], x):
        hs = mx.linear(rows, q1)
        assert_product(hs, ref_round(rows), ref_round(n1))
        hs = torch.relu(hs)
        assert_product(mx.linear(hs, q2), ref_round(hs), ref_round(n2))


@pytest.mark.parametrize("m,n,k", [(1, 1000, 4096), (8, 200, 30000), (40, 300, 5000), (200, 500, 3000), (600, 700, 500), (100, 300, 16384)])
def test_results_repeat_bit_for_bit(mx, m, n, k):
    x, w = values(m, k, BF16, 1), mx.quantize(values(n, k, BF16, 2))
    first = mx.linear(x, w)
    for _ in range(5):
        assert torch.equal(mx.linear(x, w), first)


@pytest.mark.parametrize("m,n,k", [(1, 1000, 4096), (8, 200, 30000), (40, 300, 5000), (300, 500, 700), (100, 130, 9000)])
def test_two_streams_and_two_graphs(mx, m, n, k):
    """Calls on two streams at once and two captured graphs replayed in turn with eager work between
    them: each has workspaces of its own."""
    w1, w2 = values(n, k, BF16, 1), values(n, k, BF16, 2)
    q1, q2 = mx.quantize(w1), mx.quantize(w2)
    x = values(m, k, BF16, 3)
    want1, want2 = mx.linear(x, q1), mx.linear(x, q2)
    wanted_grad = mx.linear_grad(want1, mx.linear_train(x, w1)[1])
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            outs.append((mx.linear(x, q1), want1))
        with torch.cuda.stream(s2):
            outs.append((mx.linear(x, q2), want2))
    torch.cuda.synchronize()
    for got, want in outs:
        assert torch.equal(got, want)
    gx = x.clone()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y1 = mx.linear(gx, q1)
        t1, saved = mx.linear_train(gx, w1)
        dx1, dw1 = mx.linear_grad(y1, saved)
    with torch.cuda.graph(g2):
        y2 = mx.linear(gx, q2)
    for r in range(4):
        xr = values(m, k, BF16, 10 + r) if r else x
        gx.copy_(xr)
        g1.replay()
        g2.replay()
        e1, e2 = mx.linear(xr, q1), mx.linear(xr, q2)
        torch.cuda.synchronize()
        assert torch.equal(y1, e1) and torch.equal(y2, e2)
        et, es = mx.linear_train(xr, w1)
        edx, edw = mx.linear_grad(e1, es)
        assert torch.equal(t1, et) and torch.equal(dx1, edx) and torch.equal(dw1, edw)
        if r == 0:
            assert torch.equal(dx1, wanted_grad[0]) and torch.equal(dw1, wanted_grad[1])


def test_offsets_past_32_bits(mx):
    """A matrix of more than 2^32 bytes, its last rows compared: quantised along and down, and back."""
    rows, k = 66000, 33000
    x = torch.zeros(rows, k, dtype=BF16, device="cuda")
    x[-40:] = values(40, k, BF16, 1)
    q = mx.quantize(x)
    tail = mx.dequantize(q, BF16)[-40:]
    assert torch.equal(tail.cpu().double(), ref_round(x[-40:]))
    down = mx.quantize(x, 0)
    last = mx.quantize(x[-(rows % 512) - 512:], 0)  # whole groups of the same rows
    assert torch.equal(down.codes[:, -last.codes.shape[1]:], last.codes) and torch.equal(down.scales[:, -2:], last.scales)
    y = mx.matmul(mx.quantize(x[-40:, :200]), mx.quantize(x[:, :200].contiguous()), BF16)
    assert_product(y[:, -40:], ref_round(x[-40:, :200]), ref_round(x[-40:, :200]))
    assert not y[:, :-40].any()


def test_first_calls_of_a_process_inside_a_capture(mx):
    """Kernels are loaded and the device asked for its size by the first call, which may be a captured one."""
    import subprocess
    import sys

    code = """
import torch
from gpumon.ops import mx
g0 = torch.Generator().manual_seed(1)
x = torch.randn(300, 260, generator=g0).to(torch.bfloat16).cuda()
w = torch.randn(400, 260, generator=g0).to(torch.bfloat16).cuda()
dy = torch.randn(300, 400, generator=g0).to(torch.bfloat16).cuda()
torch.cuda.synchronize()
def step():
    y, saved = mx.linear_train(x, w)
    dx, dw = mx.linear_grad(dy, saved)
    q = mx.quantize(w)
    return [y, dx, dw, mx.linear(x[:1], q), mx.linear(x[:20], q), mx.dequantize(q), mx.matmul(q, q)]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = step()
want = step()
for _ in range(3):
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
print("ok")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr[-2000:]


def test_two_threads_at_once(mx):
    import threading

    xs = [values(200 + 30 * i, 700, BF16, i) for i in range(2)]
    w = mx.quantize(values(300, 700, BF16, 9))
    want = [mx.linear(x, w) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                y = mx.linear(xs[i], w)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(y, want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_one_tensor_in_both_places(mx):
    x = values(90, 200, BF16, 1)
    v = ref_round(x)
    q = mx.quantize(x)
    assert_product(mx.matmul(q, q, F32), v, v)
    y, saved = mx.linear_train(x, x)
    dx, dw = mx.linear_grad(y, saved)
    assert_product(y, v, v)
    assert_product(dx, ref_round(y), ref_round(x.t()))
    assert_product(dw, ref_round(y.t()), ref_round(x.t()))


def test_training_step_with_nan_and_infinities(mx):
    x, w, dy = values(70, 130, BF16, 1, True), values(50, 130, F32, 2, True), values(70, 50, BF16, 3, True)
    y, saved = mx.linear_train(x, w)
    dx, dw = mx.linear_grad(dy, saved)
    assert_product(y, ref_round(x), ref_round(w))
    assert_product(dx, ref_round(dy), ref_round(w.t()))
    assert_product(dw, ref_round(dy.t()), ref_round(x.t()))


def test_views_that_share_or_negate_their_elements(mx):
    base = values(1, 700, BF16, 2)
    w = values(60, 200, BF16, 3)
    wq, wv = mx.quantize(w), ref_round(w)
    for x in (base[:, :200].expand(40, 200), base.as_strided((40, 200), (3, 1)), base.as_strided((40, 200), (1, 3)),
              base.as_strided((40, 200), (0, 0)), torch._neg_view(values(40, 200, BF16, 4))):
        assert_quantized(mx.quantize(x), x)
        assert_quantized(mx.quantize(x, 0), x.t())
        assert_product(mx.linear(x, wq), ref_round(x), wv)
        y, saved = mx.linear_train(x, w)
        assert_product(y, ref_round(x), wv)
        dy = x[:, :60]
        dx, dw = mx.linear_grad(dy, saved)
        assert_product(dx, ref_round(dy), ref_round(w.t()))
        assert_product(dw, ref_round(dy.t()), ref_round(x.t()))


def test_nothing_to_do(mx):
    q0, q = mx.quantize(torch.empty(0, 70, device="cuda")), mx.quantize(values(5, 70, F32, 1))
    assert mx.dequantize(q0).shape == (0, 70)
    assert mx.matmul(q0, q).shape == (0, 5) and mx.matmul(q, q0).shape == (5, 0)
    assert mx.linear(values(3, 70, BF16, 1), q0).shape == (3, 0)
    assert mx.linear(torch.empty(2, 0, 70, device="cuda"), q).shape == (2, 0, 5)
    for bad in (lambda: mx.quantize(torch.empty(4, 0, device="cuda")), lambda: mx.quantize(torch.empty(0, 4, device="cuda"), 0),
                lambda: mx.quantize_both(torch.empty(0, 4, device="cuda")),
                lambda: mx.linear_train(values(3, 4, BF16), torch.empty(0, 4, dtype=BF16, device="cuda"))):
        with pytest.raises(ValueError):
            bad()


def test_refusals_on_the_gpu(mx):
    x, w = values(3, 70, BF16, 1), values(5, 70, BF16, 2)
    q = mx.quantize(w)
    for bad in (lambda: mx.quantize(x[0]), lambda: mx.quantize(x, 2), lambda: mx.linear(x[:, :69], q),
                lambda: mx.linear(values(1, 1, BF16)[0, 0], q), lambda: mx.matmul(q, mx.quantize(x[:, :69])),
                lambda: mx.linear_train(x, w[:, :69]), lambda: mx.linear_grad(x, mx.linear_train(x, w)[1])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: mx.quantize(x.double()), lambda: mx.linear(x.int(), q), lambda: mx.linear(x, w),
                lambda: mx.linear_grad(values(3, 5, F16), mx.linear_train(x, w)[1])):
        with pytest.raises(TypeError):
            bad()


def test_weights_dropped_while_another_stream_uses_them(mx):
    """record_stream: memory of a quantised matrix is not given out again before the other stream is done."""
    x = values(64, 4096, BF16, 1)
    w = values(4096, 4096, BF16, 2)
    want = mx.linear(x, mx.quantize(w))
    s = torch.cuda.Stream()
    for _ in range(5):
        q = mx.quantize(w)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(10):
                y = mx.linear(x, q)
        q.record_stream(s)
        del q
        torch.empty(9 << 20, dtype=torch.uint8, device="cuda").fill_(255)
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_products_past_32_bits(mx):
    """Operands and results of more than 2^32 bytes, with whole numbers so that every sum is exact."""
    g = torch.Generator(device="cuda").manual_seed(7)

    def whole(rows, k):
        v = torch.randint(-3, 4, (rows, k), generator=g, device="cuda").to(BF16)
        v[:, ::32] = 6  # one scale everywhere
        return v

    n, k = 66000, 135000  # 4.5e9 bytes of codes
    w = torch.zeros(n, k, dtype=BF16, device="cuda")
    w[:64], w[-64:] = whole(64, k), whole(64, k)
    q = mx.quantize(w)
    ends = torch.cat([w[:64], w[-64:]]).float()
    del w
    for m in (1, 5, 40, 200):
        x = whole(m, k)
        y = mx.matmul(mx.quantize(x), q, F32)
        assert torch.equal(torch.cat([y[:, :64], y[:, -64:]], 1), x.float() @ ends.t()), m
        assert not y[:, 64:-64].any()
        if m in (1, 40):
            assert torch.equal(mx.linear(x.float(), q)[:, -64:], y[:, -64:])
    del q, y
    m, n, k = 70000, 33000, 64  # 4.6e9 bytes of results
    a, b = whole(m, k), whole(n, k)
    y = mx.matmul(mx.quantize(a), mx.quantize(b), F32)
    for rows in (slice(0, 300), slice(35000, 35200), slice(m - 300, m)):
        assert torch.equal(y[rows], a[rows].float() @ b.float().t())


def test_copied_and_loaded_matrices_and_saved_layers(mx):
    """Copies that outlive what they were made from, whose memory holds something else by then."""
    import copy
    import io

    x, w = torch.randn(5, 300, device="cuda").bfloat16(), torch.randn(70, 300, device="cuda").bfloat16()
    dy = torch.randn(5, 70, device="cuda").bfloat16()
    q = mx.quantize(w)
    y, (want, saved) = mx.linear(x, q), mx.linear_train(x, w)
    grads = mx.linear_grad(dy, saved)
    file = io.BytesIO()
    torch.save((q, saved), file)
    file.seek(0)
    copies = [copy.deepcopy((q, saved)), torch.load(file, weights_only=False)]
    q.buf.fill_(255)
    saved.buf.fill_(255)
    del q
    for cq, cs in copies:
        assert torch.equal(mx.linear(x, cq), y)
        for a, b in zip(mx.linear_grad(dy, cs), grads):
            assert torch.equal(a, b)
    cs.buf = cs.buf.cpu()
    with pytest.raises(ValueError, match="saved is on cpu"):
        mx.linear_grad(dy, cs)
