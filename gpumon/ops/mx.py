"""MXFP4 operators on GPU tensors: quantisation, product, linear layer and its training step.

What a node that serves or trains in 4 bits runs on the matrix path that
``gpu_mfma_tflops{dtype="f6f4"}`` counts, as hand-written gfx950 kernels (``csrc/hip/mx_quant.hip``,
``csrc/hip/mx_product.hip``; format and layout: ``csrc/hip/mx.h``). ``gpumon load --kind mxlinear``
drives the card with the linear layer on quantised weights; the training step is for programs that call it.

An MXFP4 matrix holds 32 consecutive elements of a row as 4-bit numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6
and their negatives) times one power of two, ``2^(floor(log2 amax) - 2)``; elements are rounded to
nearest, halves to the even code, and end at 6. A block with a NaN or an infinity stands for NaN.

* :func:`quantize` / :func:`quantize_both` / :func:`dequantize` — to the format and back.
* :func:`matmul` — ``a @ b.T`` of two quantised matrices, f32 sums.
* :func:`linear` — unquantised rows on quantised weights (serving: single tokens to prompts).
* :func:`linear_train` / :func:`linear_grad` — the layer's training step, all three products in 4 bits.

Tensors are bf16, f16 or f32 on one GPU; work goes to that device's current torch stream and can be
captured into a graph (workspaces come from torch's allocator, so each graph has its own). Results
carry no autograd graph: :func:`linear_grad` is the backward pass, and where a gradient would be lost
(an input of the linear layer that requires one while they are recorded, or has a tangent) the call is
refused; under ``torch.no_grad()``, as in the forward pass of a ``torch.autograd.Function``, it is not.
Errors of arguments are ``ValueError`` / ``TypeError``, before anything is launched.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from .._native import hip as _load_hip

DTYPES = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
BLOCK = 32


hip = functools.cache(_load_hip)  # looked up once: an import statement's search costs as much as a launch


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    def _stream(device) -> int:  # noqa: F811 - the same handle without a Stream object (1.8 us of a 10 us call)
        return torch._C._cuda_getCurrentRawStream(device.index)


def _check(t, name: str, ndim=None):
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in DTYPES and (ndim is None or t.dim() == ndim):
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"mx: {name} must be a tensor, not {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"mx: {name} must be on a GPU, it is on {t.device}")
    if t.dtype not in DTYPES:
        raise TypeError(f"mx: {name} is {t.dtype}: one of bfloat16, float16, float32")
    raise ValueError(f"mx: {name} has {t.dim()} dimensions, expected {ndim}")


def _check_constant(t, name: str):
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"mx: {name} requires a gradient, which the result would not carry: detach it, or call under "
                         "torch.no_grad() and take linear_train's gradients from linear_grad")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"mx: {name} has a tangent, which the result would not carry")


def _check_dtype(dtype):
    if dtype not in DTYPES:
        raise TypeError(f"mx: dtype {dtype}: one of bfloat16, float16, float32")


def _rows(x):
    """``(x, row stride)`` of a 2-D x with its elements next to each other along a row and no overlapping
    rows (else of a copy)."""
    if x.is_neg():  # a lazily negated view: its memory holds other values
        x = x.resolve_neg()
    r, c = x.shape
    s0, s1 = x.stride()
    if (s1 == 1 or c == 1) and s0 >= c:
        return x, s0
    if r == 1 and (s1 == 1 or c == 1):
        return x, c
    x = x.contiguous()
    return x, max(x.stride(0), c)


class MxTensor:
    """A quantised matrix, ``rows`` x ``k`` with blocks along ``k``, in the kernels' order (views of one
    buffer): ``codes`` [ceil(rows/16), ceil(k/128), 4 blocks, 16 rows, 16] uint8 and ``scales``
    [ceil(rows/16), ceil(k/512), 4 blocks, 16 rows, 4 quads of blocks] uint8; zeros fill both up.
    :meth:`parts` / :meth:`pack` are the row-major form."""

    __slots__ = ("buf", "rows", "k", "device", "_codes", "_scales")

    def __init__(self, rows: int, k: int, device):
        if rows < 0 or k < 1:
            raise ValueError(f"mx: a quantised matrix needs rows >= 0 and k >= 1, not {rows} x {k}")
        rb = (rows + 15) // 16
        codes = rb * ((k + 127) // 128) * 1024
        self._hold(torch.empty(codes + rb * ((k + 511) // 512) * 256, dtype=torch.uint8, device=device), rows, k, codes)

    def _hold(self, buf, rows: int, k: int, codes: int):
        self.rows, self.k, self.buf, self.device = rows, k, buf, buf.device
        self._codes = at = buf.data_ptr()
        self._scales = at + codes

    def __reduce__(self):  # a copied or loaded matrix has its addresses from its own buffer
        return _remake, (self.buf, self.rows, self.k)

    @property
    def shape(self):
        return (self.rows, self.k)

    @property
    def codes(self):
        return self.buf[:self._scales - self._codes].view(-(-self.rows // 16), -(-self.k // 128), 4, 16, 16)

    @property
    def scales(self):
        return self.buf[self._scales - self._codes:].view(-(-self.rows // 16), -(-self.k // 512), 4, 16, 4)

    @staticmethod
    def pack(codes, scales, k: int) -> "MxTensor":
        """From row-major parts on a GPU: codes [rows, ceil(k/32)*16] uint8 (the even element in the low
        nibble), scales [rows, ceil(k/32)] uint8 (exponent + 127; 255: NaN). Elements past k are ignored."""
        blocks = -(-k // BLOCK)
        for t, name, width in ((codes, "codes", blocks * 16), (scales, "scales", blocks)):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8:
                raise TypeError(f"mx: {name} must be a uint8 tensor")
            if not t.is_cuda:
                raise ValueError(f"mx: {name} must be on a GPU, it is on {t.device}")
            if t.dim() != 2 or t.shape[1] != width or t.shape[0] != codes.shape[0]:
                raise ValueError(f"mx: {name} is {tuple(t.shape)}, expected ({codes.shape[0]}, {width}) for k = {k}")
        if codes.device != scales.device:
            raise ValueError(f"mx: codes are on {codes.device}, scales on {scales.device}")
        q = MxTensor(codes.shape[0], k, codes.device)
        rb, quads, groups = -(-q.rows // 16), -(-k // 128), -(-k // 512)
        full = codes.new_zeros(rb * 16, quads * 64)
        full[:q.rows, :(k + 1) // 2] = codes[:, :(k + 1) // 2]
        if k % 2:
            full[:, k // 2] &= 15
        q.codes.copy_(full.view(rb, 16, quads, 4, 16).permute(0, 2, 3, 1, 4))
        full = scales.new_zeros(rb * 16, groups * 16)
        full[:q.rows, :blocks] = scales
        q.scales.copy_(full.view(rb, 16, groups, 4, 4).permute(0, 2, 4, 1, 3))
        return q

    def parts(self):
        """(codes, scales) row-major, as :meth:`pack` takes them."""
        blocks, r16 = -(-self.k // BLOCK), -(-self.rows // 16) * 16
        codes = self.codes.permute(0, 3, 1, 2, 4).reshape(r16, -(-self.k // 128) * 64)[:self.rows, :blocks * 16]
        scales = self.scales.permute(0, 3, 1, 4, 2).reshape(r16, -(-self.k // 512) * 16)[:self.rows, :blocks]
        return codes.contiguous(), scales.contiguous()

    def record_stream(self, stream) -> None:
        """As ``torch.Tensor.record_stream``: before it is dropped while work on another stream uses it."""
        self.buf.record_stream(stream)

    def __repr__(self):
        return f"MxTensor({self.rows} x {self.k}, {self.device})"


def _remake(buf, rows: int, k: int) -> MxTensor:
    rb = (rows + 15) // 16
    codes, scales = rb * ((k + 127) // 128) * 1024, rb * ((k + 511) // 512) * 256
    if buf.dtype != torch.uint8 or buf.shape != (codes + scales,) or not buf.is_contiguous():
        raise ValueError(f"mx: a {rows} x {k} matrix needs a buffer of {codes + scales} uint8, not {tuple(buf.shape)} {buf.dtype}")
    q = MxTensor.__new__(MxTensor)
    q._hold(buf, rows, k, codes)
    return q


def _check_mx(q, name: str):
    if not isinstance(q, MxTensor):
        raise TypeError(f"mx: {name} must be an MxTensor, not {type(q).__name__}")


def _check_gpu(q, name: str):
    if not q.buf.is_cuda:
        raise ValueError(f"mx: {name} must be on a GPU, it is on {q.device}")


def quantize(x, axis: int = 1) -> MxTensor:
    """x [r, c] with blocks along its rows (``axis`` 1 or -1: r x c) or down its columns (``axis`` 0 or
    -2: c x r, the transposed matrix, as a product that contracts over r takes it)."""
    _check(x, "x", 2)
    if axis not in (0, 1, -1, -2):
        raise ValueError(f"mx: axis {axis}: 0 or 1")
    down = axis in (0, -2)
    if x.stride(0) == 1 and x.stride(1) >= x.shape[0] > 1:  # a transposed view: the other direction of its base
        x, down = x.t(), not down
    x, stride = _rows(x)
    r, c = x.shape
    dev = x.device
    q = MxTensor(c, r, dev) if down else MxTensor(r, c, dev)
    if q.rows:
        hip().mx_quantize(dev.index, x.data_ptr(), DTYPES[x.dtype], r, c, stride, down, q._codes, q._scales, _stream(dev))
    return q


def quantize_both(x):
    """``(quantize(x, 1), quantize(x, 0))`` from one reading of x."""
    _check(x, "x", 2)
    swap = x.stride(0) == 1 and x.stride(1) >= x.shape[0] > 1
    x, stride = _rows(x.t() if swap else x)
    r, c = x.shape
    dev = x.device
    along, down = MxTensor(r, c, dev), MxTensor(c, r, dev)
    hip().mx_quantize_both(dev.index, x.data_ptr(), DTYPES[x.dtype], r, c, stride, along._codes, along._scales,
                           down._codes, down._scales, _stream(dev))
    return (down, along) if swap else (along, down)


def dequantize(q: MxTensor, dtype=torch.float32):
    """What q stands for, [rows, k]; exact in bf16 and f32, rounded in f16."""
    _check_mx(q, "q")
    _check_dtype(dtype)
    _check_gpu(q, "q")
    out = torch.empty(q.rows, q.k, dtype=dtype, device=q.device)
    if q.rows:
        hip().mx_dequantize(q.device.index, q._codes, q._scales, q.rows, q.k, out.data_ptr(), DTYPES[dtype], q.k,
                            _stream(q.device))
    return out


def matmul(a: MxTensor, b: MxTensor, dtype=torch.bfloat16):
    """a [m, k] @ b [n, k].T in ``dtype``: sums in 32 bits, rounded once."""
    _check_mx(a, "a")
    _check_mx(b, "b")
    _check_dtype(dtype)
    if a.k != b.k:
        raise ValueError(f"mx: a is {a.rows} x {a.k} and b {b.rows} x {b.k}: the second sizes differ")
    if a.device != b.device:
        raise ValueError(f"mx: a is on {a.device}, b on {b.device}")
    _check_gpu(a, "a")
    c = torch.empty(a.rows, b.rows, dtype=dtype, device=a.device)
    if c.numel():
        h, dev = hip(), a.device.index
        need = h.mx_product_workspace(a.rows, b.rows, a.k)
        ws = torch.empty(need, dtype=torch.uint8, device=a.device) if need else None
        h.mx_product(dev, a._codes, a._scales, b._codes, b._scales, a.rows, b.rows, a.k, c.data_ptr(), DTYPES[dtype],
                     b.rows, ws.data_ptr() if need else 0, need, _stream(a.device))
    return c


def linear(x, w: MxTensor):
    """x [..., k] on weights w (n x k): x quantised along k, times w.T; [..., n] in x's type."""
    _check(x, "x")
    _check_constant(x, "x")
    _check_mx(w, "w")
    if x.dim() < 1 or x.shape[-1] != w.k:
        raise ValueError(f"mx: x is {tuple(x.shape)}, its last size must be the weights' k = {w.k}")
    if x.device != w.device:
        raise ValueError(f"mx: x is on {x.device}, w on {w.device}")
    flat = x.dim() == 2
    x2, stride = _rows(x if flat else x.reshape(-1, w.k))
    m, n, dev = x2.shape[0], w.rows, x.device
    y = torch.empty((m, n) if flat else (*x.shape[:-1], n), dtype=x.dtype, device=dev)
    if m and n:
        h, dtype = hip(), DTYPES[x.dtype]
        need = h.mx_linear_workspace(m, n, w.k, dtype)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        h.mx_linear(dev.index, x2.data_ptr(), dtype, stride, w._codes, w._scales, m, n, w.k, y.data_ptr(), n,
                    ws.data_ptr() if need else 0, need, _stream(dev))
    return y


class LinearSaved:
    """What :func:`linear_train` keeps for :func:`linear_grad`: x and w with blocks along the axes that
    the gradients contract over."""

    __slots__ = ("buf", "shape", "rows", "n", "k", "dtype", "w_dtype", "device")

    def record_stream(self, stream) -> None:
        """As ``torch.Tensor.record_stream``."""
        if self.buf is not None:
            self.buf.record_stream(stream)


def linear_train(x, w):
    """Forward pass with x [..., k] and w [n, k] both quantised here: ``(y [..., n], saved)``."""
    _check(x, "x")
    _check(w, "w", 2)
    _check_constant(x, "x")
    _check_constant(w, "w")
    if x.dim() < 1 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"mx: x is {tuple(x.shape)}, w {tuple(w.shape)}: the last sizes differ")
    if x.device != w.device:
        raise ValueError(f"mx: x is on {x.device}, w on {w.device}")
    n, k = w.shape
    if n < 1 or k < 1:
        raise ValueError(f"mx: w is {tuple(w.shape)}: neither size may be 0")
    dev = x.device
    x2, x_stride = _rows(x if x.dim() == 2 else x.reshape(-1, k))
    w, w_stride = _rows(w)
    m = x2.shape[0]
    saved = LinearSaved()
    saved.shape, saved.rows, saved.n, saved.k = x.shape, m, n, k
    saved.dtype, saved.w_dtype, saved.device = x.dtype, w.dtype, dev
    y = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=dev)
    if m == 0:
        saved.buf = None
        return y, saved
    h = hip()
    size, need = h.mx_linear_train_saved(m, n, k), h.mx_linear_train_workspace(m, n, k)
    saved.buf = torch.empty(size, dtype=torch.uint8, device=dev)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    h.mx_linear_train(dev.index, x2.data_ptr(), DTYPES[x.dtype], x_stride, w.data_ptr(), DTYPES[w.dtype], w_stride, m,
                      n, k, y.data_ptr(), n, saved.buf.data_ptr(), size, ws.data_ptr(), need, _stream(dev))
    return y, saved


def linear_grad(dy, saved: LinearSaved, need_dx: bool = True, need_dw: bool = True):
    """Backward pass: ``(dx, dw)`` in x's and w's type (None where not needed). Straight-through: the
    gradients of the layer as if quantising were the identity, each product in 4 bits with dy
    quantised along the axis that it contracts over. Neither's bits depend on whether the other is needed."""
    _check(dy, "dy")
    _check_constant(dy, "dy")
    if not isinstance(saved, LinearSaved):
        raise TypeError(f"mx: saved must come from linear_train, not {type(saved).__name__}")
    m, n, k, dev = saved.rows, saved.n, saved.k, saved.device
    if dy.shape[:-1] != saved.shape[:-1] or dy.dim() < 1 or dy.shape[-1] != n:
        raise ValueError(f"mx: dy is {tuple(dy.shape)}, expected {tuple(saved.shape[:-1]) + (n,)}")
    if dy.dtype != saved.dtype:
        raise TypeError(f"mx: dy is {dy.dtype}, the layer's output {saved.dtype}")
    if dy.device != dev:
        raise ValueError(f"mx: dy is on {dy.device}, the layer on {dev}")
    if m and saved.buf.device != dev:  # loaded from a file to somewhere else
        raise ValueError(f"mx: saved is on {saved.buf.device}, the layer on {dev}")
    dx = torch.empty(saved.shape, dtype=saved.dtype, device=dev) if need_dx else None
    if m == 0:
        return dx, torch.zeros(n, k, dtype=saved.w_dtype, device=dev) if need_dw else None
    dw = torch.empty(n, k, dtype=saved.w_dtype, device=dev) if need_dw else None
    if need_dx or need_dw:
        h = hip()
        d2, stride = _rows(dy if dy.dim() == 2 else dy.reshape(-1, n))
        need = h.mx_linear_grad_workspace(m, n, k)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        h.mx_linear_grad(dev.index, d2.data_ptr(), DTYPES[dy.dtype], stride, saved.buf.data_ptr(), m, n, k,
                         dx.data_ptr() if need_dx else 0, k, dw.data_ptr() if need_dw else 0, DTYPES[saved.w_dtype], k,
                         ws.data_ptr(), need, _stream(dev))
    return dx, dw
