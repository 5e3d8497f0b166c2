"""Products of matrices in 8-bit floating point with a float32 scale for each block of 128 (or 128 x 128), for PyTorch:
`quantize_fp8`, `matmul_fp8` and the differentiable `linear_fp8`.

    values, scales = quantize_fp8(x)                        # a scale for 128 values of a row
    weight = quantize_fp8(w, block=(128, 128))              # a scale for each 128 x 128
    y = matmul_fp8(values, scales, *weight)                 # x @ w.mT, in bfloat16 unless asked otherwise

A block of 128 along k is multiplied on the tensor cores, its product scaled and added in float32; the result is rounded
once. Calls take CUDA tensors and enqueue on torch's current stream of the tensors' device.
"""
import math
import struct

import torch
from torch import Tensor

from . import _lib
from ._eager import direct

__all__ = ["quantize_fp8", "matmul_fp8", "linear_fp8"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_KINDS = {torch.float8_e4m3fn: 3, torch.float8_e5m2: 4}
_OPERAND = struct.Struct("=2Q2Q2I")


def _fail(name, message, kind=ValueError):
    raise kind(f"metal_linalg_torch.{name}: {message}")


def _on_gpu(name, what, x):
    if not isinstance(x, Tensor):
        _fail(name, f"{what} must be a tensor, got {type(x).__name__}", TypeError)
    if not x.is_cuda and not x.is_meta:
        _fail(name, f"tensors on {x.device} are not supported; use CUDA (this library has no CPU path)")


def _padded(x, lead, rows, cols, dtype):
    """An uninitialised [..., rows, cols] on x's device whose rows lie a multiple of 16 bytes apart."""
    wide = -(-cols // 16) * 16
    values = x.new_empty((*lead, rows, wide), dtype=dtype)
    return values if wide == cols else values[..., :cols]


def _quantize(x, block_rows, transpose, dtype):
    *lead, m, n = x.shape
    if len(lead) > 1 and x.numel():
        x = x.reshape(-1, m, n)                         # copies only what no strides can describe
    *outer, rows, cols = x.stride()
    if transpose:
        m, n, rows, cols = n, m, cols, rows
    values = _padded(x, lead, m, n, dtype)
    scales = x.new_empty((*lead, -(-m // block_rows), -(-n // 128)), dtype=torch.float32)
    if not values.numel():
        return values, scales
    # a dimension of one may carry any stride: it is given one the library can read along
    if n == 1:
        cols = 1
    elif m == 1 and cols != 1:
        rows = 1
    elif rows != 1 and cols != 1:
        x = x.contiguous()
        *outer, rows, cols = x.stride()
        if transpose:
            rows, cols = cols, rows
    batch, across = (x.shape[0], outer[0]) if outer else (1, 0)
    device = _lib.use_stream_of(x)
    _lib.check(_lib.lib.metal_linalg_quantize_fp8(x.data_ptr(), _DTYPES[x.dtype], batch, m, n, across, rows, cols, block_rows,
                                                  _KINDS[dtype], values.data_ptr(), -(-n // 16) * 16, scales.data_ptr(), device))
    return values, scales


@torch.library.custom_op("metal_linalg::quantize_fp8", mutates_args=())
def _quantize_op(x: Tensor, block_rows: int, transpose: bool, dtype: torch.dtype) -> tuple[Tensor, Tensor]:
    return _quantize(x, block_rows, transpose, dtype)


@_quantize_op.register_fake
def _(x, block_rows, transpose, dtype):
    *lead, m, n = x.mT.shape if transpose else x.shape
    wide = -(-n // 16) * 16
    return (x.new_empty((*lead, m, wide), dtype=dtype)[..., :n],
            x.new_empty((*lead, -(-m // block_rows), -(-n // 128)), dtype=torch.float32))


def quantize_fp8(x, *, block=(1, 128), transpose=False, dtype=torch.float8_e4m3fn):
    """``x`` [..., M, N] (float32, bfloat16 or float16) in 8-bit floating point: ``(values, scales)``.

    ``block`` is (1, 128) or (128, 128): a float32 scale for that many neighbours, ``max|x| / M`` (M: the largest value of
    ``dtype``, 448 or 57344; at least 2 ** -126), and values ``x / scale`` (in float32) rounded to the nearest, ties to even.
    ``scales`` is [..., ceil(M / block[0]), ceil(N / 128)]; ``values`` is [..., M, N] with its rows a multiple of 16
    bytes apart, as `matmul_fp8` reads them. With ``transpose`` the last two dimensions of x are exchanged first (without a
    copy). Strides are taken as they are where one of the last two dimensions is contiguous. A block with a NaN or an
    infinity stands for NaN throughout. Not differentiable (gradients pass through `linear_fp8`).
    """
    name = "quantize_fp8"
    _on_gpu(name, "x", x)
    if x.dtype not in _DTYPES:
        _fail(name, f"x must be float32, bfloat16 or float16, got {x.dtype}", TypeError)
    if dtype not in _KINDS:
        _fail(name, f"dtype must be torch.float8_e4m3fn or torch.float8_e5m2, got {dtype}", TypeError)
    if tuple(block) not in ((1, 128), (128, 128)):
        _fail(name, f"block must be (1, 128) or (128, 128), got {tuple(block)}")
    if x.dim() < 2:
        _fail(name, f"expected a tensor of shape [..., M, N], got shape {tuple(x.shape)}")
    if torch.is_grad_enabled() and x.requires_grad:
        _fail(name, "not differentiable; use linear_fp8, or detach x", RuntimeError)
    if not direct(name, x):
        return torch.ops.metal_linalg.quantize_fp8(x, block[0], bool(transpose), dtype)
    return _quantize(x, block[0], transpose, dtype)


def _block_rows(name, what, rows, scales_rows):
    if scales_rows == rows:
        return 1
    if scales_rows == -(-rows // 128):
        return 128
    _fail(name, f"{what}_scale must have {rows} or {-(-rows // 128)} rows, got {scales_rows}")


def _check_product(name, a, a_scale, b, b_scale):
    """Refuses operands that do not fit; returns the rows of their scales' blocks."""
    for what, x in (("a", a), ("a_scale", a_scale), ("b", b), ("b_scale", b_scale)):
        _on_gpu(name, what, x)
    device = a.device
    if a_scale.device != device or b.device != device or b_scale.device != device:
        _fail(name, f"a, a_scale, b and b_scale must be on one device, got {device}, {a_scale.device}, {b.device} and {b_scale.device}")
    if a.dtype not in _KINDS or b.dtype not in _KINDS:
        _fail(name, f"a and b must be float8_e4m3fn or float8_e5m2, got {a.dtype} and {b.dtype}", TypeError)
    if a_scale.dtype != torch.float32 or b_scale.dtype != torch.float32:
        _fail(name, f"the scales must be float32, got {a_scale.dtype} and {b_scale.dtype}", TypeError)
    sizes, others = a.shape, b.shape
    if len(sizes) < 2 or len(others) < 2 or sizes[-1] != others[-1] or (len(others) > 2 and others[:-2] != sizes[:-2]):
        _fail(name, f"expected a [..., M, K] and b [..., N, K] or [N, K], got {tuple(sizes)} and {tuple(others)}")
    blocks = -(-sizes[-1] // 128)
    rows = []
    for what, x, s in (("a", sizes, a_scale.shape), ("b", others, b_scale.shape)):
        if len(s) != len(x) or s[:-2] != x[:-2] or s[-1] != blocks:
            _fail(name, f"expected {what}_scale [..., rows, {blocks}] for {tuple(x)}, got {tuple(s)}")
        rows.append(_block_rows(name, what, x[-2], s[-2]))
    return rows


def _operand(x, scale, block_rows, batched):
    """A metal_linalg_fp8_operand as bytes, and the tensors it points to. What the library cannot read in place (rows that
    are not a multiple of 16 bytes apart, say) is copied once."""
    *_, m, k = x.shape
    *outer, stride, one = x.stride()
    if m == 1:
        stride = -(-k // 16) * 16                       # any stride will do
    across = outer[0] if batched else 0
    at = x.data_ptr()
    if (one != 1 and k > 1) or stride < k or stride % 16 or at % 16 or (batched and (across % stride or across < stride * m)):
        copy = _padded(x, x.shape[:-2], m, k, x.dtype)
        copy.copy_(x)
        x, at, stride = copy, copy.data_ptr(), -(-k // 16) * 16
        across = stride * m if batched else 0
    scale = scale.contiguous()
    return _OPERAND.pack(at, scale.data_ptr(), stride, across, _KINDS[x.dtype], block_rows), (x, scale)


def _matmul(a, a_scale, b, b_scale, a_rows, b_rows, out_dtype):
    *lead, m, k = a.shape
    n = b.shape[-2]
    out = a.new_empty((*lead, m, n), dtype=out_dtype)
    if not (m and n and k) or not out.numel():
        return out.zero_()
    batch = 1
    if lead:
        batch = out.numel() // (m * n)
        if len(lead) > 1:
            a = a.reshape(-1, m, k)
            if b.dim() > 2:
                b = b.reshape(-1, n, k)
        if b.dim() == 2 and a_rows == 1 and a.stride(0) == m * a.stride(1):
            a, m, batch = a.flatten(0, 1), batch * m, 1      # one matrix for the whole batch: the rows behind one another
    pa, keep_a = _operand(a, a_scale, a_rows, batch > 1)
    pb, keep_b = _operand(b, b_scale, b_rows, batch > 1 and b.dim() == 3)
    device = _lib.use_stream_of(out)
    _lib.check(_lib.lib.metal_linalg_matmul_fp8(pa, pb, batch, m, n, k, out.data_ptr(), _DTYPES[out_dtype], device))
    return out


@torch.library.custom_op("metal_linalg::matmul_fp8", mutates_args=())
def _matmul_op(a: Tensor, a_scale: Tensor, b: Tensor, b_scale: Tensor, a_rows: int, b_rows: int, out_dtype: torch.dtype) -> Tensor:
    return _matmul(a, a_scale, b, b_scale, a_rows, b_rows, out_dtype)


@_matmul_op.register_fake
def _(a, a_scale, b, b_scale, a_rows, b_rows, out_dtype):
    return a.new_empty((*a.shape[:-1], b.shape[-2]), dtype=out_dtype)


def matmul_fp8(a, a_scale, b, b_scale, *, out_dtype=torch.bfloat16):
    """``a @ b.mT`` of two matrices (or batches of them) in 8-bit floating point, each with a scale for every block of 128
    along k: ``a`` [..., M, K] and ``b`` [..., N, K], or [N, K] for a whole batch, in float8_e4m3fn or float8_e5m2
    (each its own); the scales [..., rows, ceil(K / 128)] in float32 with a row for every row of the operand, or for every 128
    (as `quantize_fp8` gives them). Returns [..., M, N] in ``out_dtype`` (float32, bfloat16 or float16), rounded once from
    float32. Operands are read in place where k is contiguous and rows lie a multiple of 16 bytes apart; others are
    copied. Not differentiable.
    """
    name = "matmul_fp8"
    a_rows, b_rows = _check_product(name, a, a_scale, b, b_scale)
    if out_dtype not in _DTYPES:
        _fail(name, f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}", TypeError)
    if torch.is_grad_enabled() and (a.requires_grad or a_scale.requires_grad or b.requires_grad or b_scale.requires_grad):
        _fail(name, "not differentiable; use linear_fp8, or detach the operands", RuntimeError)
    if not direct(name, a, a_scale, b, b_scale):
        return torch.ops.metal_linalg.matmul_fp8(a, a_scale, b, b_scale, a_rows, b_rows, out_dtype)
    return _matmul(a, a_scale, b, b_scale, a_rows, b_rows, out_dtype)


def _product(quantize, matmul, x, y, x_block, y_block, x_turned, y_turned, out_dtype):
    """Both quantised and multiplied: a scale for 128 along the summed dimension, rows of 1 or 128."""
    e4m3 = torch.float8_e4m3fn
    return matmul(*quantize(x, x_block, x_turned, e4m3), *quantize(y, y_block, y_turned, e4m3), x_block, y_block, out_dtype)


def _linear_grads(ctx, dy, quantize=None, matmul=None):
    x, w = ctx.saved_tensors
    if quantize is None or not direct("linear_fp8", dy, x, w):
        quantize, matmul = torch.ops.metal_linalg.quantize_fp8, torch.ops.metal_linalg.matmul_fp8
    dx = dw = None
    dy = dy.to(x.dtype)
    if ctx.needs_input_grad[0]:
        dx = _product(quantize, matmul, dy, w, 1, 128, False, True, x.dtype)
    if ctx.needs_input_grad[1]:
        dw = _product(quantize, matmul, dy, x, 1, 1, True, True, w.dtype)
    return dx, dw


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return _product(_quantize, _matmul, x, w, 1, 128, False, False, x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return _linear_grads(ctx, dy, _quantize, _matmul)


@torch.library.custom_op("metal_linalg::linear_fp8", mutates_args=())
def _linear_op(x: Tensor, w: Tensor) -> Tensor:
    return _product(_quantize, _matmul, x, w, 1, 128, False, False, x.dtype)


@_linear_op.register_fake
def _(x, w):
    return x.new_empty((x.shape[0], w.shape[0]))


_linear_op.register_autograd(_linear_grads, setup_context=lambda ctx, inputs, output: ctx.save_for_backward(*inputs))


def linear_fp8(x, w):
    """``x @ w.mT`` with both operands in 8-bit floating point (e4m3), differentiable: ``x`` [..., K] and ``w`` [N, K] in
    float32, bfloat16 or float16 (each its own type) give [..., N] in x's type.

    x is quantised with a scale for 128 values of a row, w with one for each 128 x 128. The gradients are the products of
    operands quantised along the dimension they are summed over: ``dx = dy @ w`` from dy's rows and w's 128 x 128
    blocks, ``dw = dy.mT @ x`` from both in blocks of 128 along the tokens. Quantisation itself counts as the identity.
    Differentiable once, not in forward mode.
    """
    name = "linear_fp8"
    _on_gpu(name, "x", x)
    _on_gpu(name, "w", w)
    if x.dtype not in _DTYPES or w.dtype not in _DTYPES:
        _fail(name, f"x and w must be float32, bfloat16 or float16, got {x.dtype} and {w.dtype}", TypeError)
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1]:
        _fail(name, f"expected x [..., K] and w [N, K], got {tuple(x.shape)} and {tuple(w.shape)}")
    if w.device != x.device:
        _fail(name, f"w is on {w.device}, x on {x.device}")
    flat = x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), x.shape[-1])
    if not direct(name, x, w):
        y = torch.ops.metal_linalg.linear_fp8(flat, w)
    elif torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        y = _Linear.apply(flat, w)
    else:
        y = _product(_quantize, _matmul, flat, w, 1, 128, False, False, x.dtype)
    return y.reshape(*x.shape[:-1], w.shape[0])
