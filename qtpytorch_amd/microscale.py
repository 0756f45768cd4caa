"""Microscaled 4-bit floating point: blocks of 32 E2M1 values along the last
dimension, each block with one power-of-two scale (E8M0).

A value is ``grid[code] * 2**(scale - 127)`` with the grid 0, 0.5, 1, 1.5, 2,
3, 4, 6 and its negatives; the scale of a block is two binades below its
largest magnitude, and a scale of 255 makes the block NaN (a block that held a NaN
or an infinity).  gfx950 multiplies such operands as they are stored, at four
times the bf16 rate, where the formats of ``mx_dtype`` (one float32 scale per
block of any length) are decoded first.

  mxfp4_quantize(x)                 -> mxfp4_tensor, rounded to nearest even
  mxfp4_tensor.dequantize(dtype)    the values
  mxfp4_matmul(a, b, bias)          a @ b.T of packed operands
  mxfp4_linear(x, weight, bias)     float x, packed on the way; differentiable

``mxfp4_linear`` passes gradients straight through the quantizer:
``dx = dy @ dequantize(weight)`` and, for a float weight, ``dw = dy.T @
dequantize(quantize(x))``, both with dy unrounded (a float32 dy below 2**-110
counts down to 2**-133) and sums in float32.  There is no forward-mode
derivative: a dual tensor is refused.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L

Tensor = torch.Tensor

_FLOATS = {torch.float32: L.MXK_IN_F32, torch.float16: L.MXK_IN_F16, torch.bfloat16: L.MXK_IN_BF16}


class mxfp4_tensor:
    """Packed values of a [..., K] tensor: ``codes`` uint8 [..., 16 * KB] (two
    a byte, the lower half first) and ``scales`` uint8 [..., KB], KB =
    ceil(K / 32); codes past K are 0."""

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes: Tensor, scales: Tensor, shape):
        shape = torch.Size(shape)
        if len(shape) < 1:
            raise ValueError("mxfp4_tensor: a tensor of at least one dimension")
        kb = -(-shape[-1] // 32)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError(f"mxfp4_tensor: codes and scales are uint8, got {codes.dtype} and {scales.dtype}")
        if codes.shape != (*shape[:-1], 16 * kb) or scales.shape != (*shape[:-1], kb):
            raise ValueError(f"mxfp4_tensor: shape {tuple(shape)} has codes [..., {16 * kb}] and scales [..., {kb}], "
                             f"got {tuple(codes.shape)} and {tuple(scales.shape)}")
        if codes.device != scales.device:
            raise L.MXKError(f"tensors on different devices: {codes.device} and {scales.device}")
        self.codes = _aligned(codes.contiguous())
        self.scales = scales.contiguous()
        self.shape = shape

    @classmethod
    def _of(cls, codes: Tensor, scales: Tensor, shape: torch.Size) -> "mxfp4_tensor":
        """Codes and scales that were allocated for this shape."""
        q = cls.__new__(cls)
        q.codes, q.scales, q.shape = codes, scales, shape
        return q

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def dim(self) -> int:
        return len(self.shape)

    def to(self, device) -> "mxfp4_tensor":
        return mxfp4_tensor(self.codes.to(device), self.scales.to(device), self.shape)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> Tensor:
        """The values as float32, float16 or bfloat16 (exact in float32 and
        bfloat16 below their largest value; float16 rounds to nearest even)."""
        dev = L.require_gpu(self.codes)
        kind = L.elem_type(dtype)
        shape = self.shape
        y = torch.empty(shape, dtype=dtype, device=dev)
        if y.numel():
            with L.on_device(dev):
                rc = L.lib().mxk_mxfp4_dequantize(self.codes.data_ptr(), self.scales.data_ptr(), _rows(shape),
                                                  shape[-1], kind, y.data_ptr(), L.stream_of(y))
            if rc:
                L.check(rc, f"mxfp4 dequantize({tuple(shape)})")
        return y

    def __repr__(self):
        return f"mxfp4_tensor(shape={tuple(self.shape)}, device={self.device})"


def _aligned(codes: Tensor) -> Tensor:
    """Codes on a 16-byte boundary, as the products read them (rows are 16-byte multiples)."""
    return codes if codes.data_ptr() % 16 == 0 else codes.clone()


def _rows(shape) -> int:
    return shape[0] if len(shape) == 2 else math.prod(shape[:-1])


def mxfp4_quantize(x: Tensor) -> mxfp4_tensor:
    """Pack a [..., K] tensor of float32, float16 or bfloat16 in blocks of 32
    along its last dimension.

    Per block: scale byte = max(exponent of the largest magnitude - 2, -127) +
    127, code = the nearest grid value of x / 2**(scale - 127), ties to the
    even code, magnitudes above 6 to 6."""
    shape = x.shape
    if len(shape) < 1:
        raise ValueError("mxfp4_quantize: a tensor of at least one dimension")
    dev = L.require_gpu(x)
    kind = _FLOATS.get(x.dtype)
    if kind is None:  # by way of float32 they would be rounded twice, or leave its range
        raise TypeError(f"mxfp4_quantize: float32, float16 or bfloat16 expected, got {x.dtype}")
    cols = ld = shape[-1]
    kb = -(-cols // 32)
    if len(shape) == 2:
        x = _row_major(x)
        ld = max(x.stride(0), cols)
        codes = torch.empty((shape[0], 16 * kb), dtype=torch.uint8, device=dev)
        scales = torch.empty((shape[0], kb), dtype=torch.uint8, device=dev)
    else:
        x = x.detach().contiguous()
        codes = torch.empty((*shape[:-1], 16 * kb), dtype=torch.uint8, device=dev)
        scales = torch.empty((*shape[:-1], kb), dtype=torch.uint8, device=dev)
    if codes.numel():
        with L.on_device(dev):
            rc = L.lib().mxk_mxfp4_quantize(x.data_ptr(), kind, _rows(shape), cols, ld, codes.data_ptr(),
                                            scales.data_ptr(), L.stream_of(codes))
        if rc:
            L.check(rc, f"mxfp4_quantize({tuple(shape)})")
    return mxfp4_tensor._of(codes, scales, shape)


def _bias_f32(bias: Optional[Tensor], shape: Tuple[int, ...]) -> Optional[Tensor]:
    if bias is None:
        return None
    if tuple(bias.shape) != shape:
        raise ValueError(f"bias of shape {shape} expected, got {tuple(bias.shape)}")
    if bias.is_complex():
        raise TypeError(f"a real bias expected, got {bias.dtype}")
    return bias.detach().float().contiguous()


def _product(a: mxfp4_tensor, b: mxfp4_tensor, rows: int, N: int, bias: Optional[Tensor], out: Tensor,
             offsets: Optional[Tensor] = None, order: Optional[Tensor] = None, top: int = 1) -> Tensor:
    """out [rows, N] = a @ b.T (+ bias), by expert where offsets are given."""
    dev = L.require_gpu(a.codes, b.codes, bias, offsets, order)
    lib = L.lib()
    a_rows, K = _rows(a.shape), b.shape[-1]
    E = 0 if offsets is None else offsets.numel() - 1
    nbytes = lib.mxk_mxfp4_matmul_workspace(a_rows, rows, N, K, E, order is not None)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with L.on_device(dev):
        rc = lib.mxk_mxfp4_matmul(a.codes.data_ptr(), a.scales.data_ptr(), a_rows, b.codes.data_ptr(),
                                  b.scales.data_ptr(), rows, N, K, L.ptr(bias), L.elem_type(out.dtype),
                                  out.data_ptr(), L.ptr(offsets), E, L.ptr(order), top, L.ptr(ws), nbytes,
                                  L.stream_of(out))
    if rc:
        L.check(rc, f"mxfp4 product({rows}x{K} by {N})")
    return out


def _row_major(x: Tensor) -> Tensor:
    """x [rows, cols] itself if its rows are contiguous (they may lie apart), else a copy."""
    return x if x.stride(1) == 1 and x.stride(0) >= x.shape[1] else x.detach().contiguous()


def _linear(x: Tensor, b: mxfp4_tensor, rows: int, bias: Optional[Tensor], offsets: Optional[Tensor] = None,
            order: Optional[Tensor] = None, top: int = 1) -> Tensor:
    """Float rows x [*, K] packed and multiplied in one call, [rows, N] of x's dtype."""
    dev = L.require_gpu(x, b.codes, bias, offsets, order)
    lib = L.lib()
    x = _row_major(x)
    N, K = b.shape[-2:]
    E = 0 if offsets is None else offsets.numel() - 1
    y = torch.empty((rows, N), dtype=x.dtype, device=dev)
    kind, stride = _FLOATS[x.dtype], max(x.stride(0), K)
    nbytes = lib.mxk_mxfp4_linear_workspace(kind, x.shape[0], stride, rows, N, K, E, order is not None)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with L.on_device(dev):
        rc = lib.mxk_mxfp4_linear(x.data_ptr(), kind, x.shape[0], stride, b.codes.data_ptr(),
                                  b.scales.data_ptr(), rows, N, K, L.ptr(bias), y.data_ptr(),
                                  L.ptr(offsets), E, L.ptr(order), top, L.ptr(ws), nbytes, L.stream_of(y))
    if rc:
        L.check(rc, f"mxfp4 linear({rows}x{K} by {N})")
    return y


def _matmul(a: mxfp4_tensor, b: mxfp4_tensor, bias: Optional[Tensor], out_dtype: torch.dtype) -> Tensor:
    out = torch.empty(*a.shape[:-1], b.shape[0], dtype=out_dtype, device=a.device)
    return _product(a, b, _rows(a.shape), b.shape[0], _bias_f32(bias, (b.shape[0],)), out)


class _MXFP4MatmulBias(torch.autograd.Function):
    """mxfp4_matmul, differentiable in its bias; the packed operands are constants."""

    @staticmethod
    def forward(ctx, bias, a, b, out_dtype):
        ctx.dtype = bias.dtype
        return _matmul(a, b, bias, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        N = dy.shape[-1]
        return _grad_bias(dy.reshape(math.prod(dy.shape[:-1]), N).contiguous(), ctx.dtype), None, None, None


def mxfp4_matmul(a: mxfp4_tensor, b: mxfp4_tensor, bias: Optional[Tensor] = None,
                 out_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """a [..., K] @ b [N, K].T (+ bias [N]) of packed operands, [..., N].
    Products are exact, sums in float32, rounded once to out_dtype.  The bias has
    a gradient, packed operands have none."""
    if not isinstance(a, mxfp4_tensor) or not isinstance(b, mxfp4_tensor):
        raise TypeError("mxfp4_matmul: two mxfp4_tensors (mxfp4_quantize packs a float tensor)")
    _no_tangents("mxfp4_matmul", bias)
    if b.dim() != 2 or a.shape[-1] != b.shape[1]:
        raise ValueError(f"mxfp4_matmul: [..., K] and [N, K] expected, got {tuple(a.shape)} and {tuple(b.shape)}")
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        return _MXFP4MatmulBias.apply(bias, a, b, out_dtype)
    return _matmul(a, b, bias, out_dtype)


def _grad(entry: str, dy: Tensor, q: mxfp4_tensor, out: Tensor, offsets: Optional[Tensor]) -> Tensor:
    dev = L.require_gpu(dy, q.codes, offsets)
    lib = L.lib()
    M, N = dy.shape
    K = q.shape[-1]
    kind = L.elem_type(dy.dtype)
    nbytes = lib.mxk_mxfp4_grad_workspace(dy.data_ptr(), kind, M, N)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with L.on_device(dev):
        rc = getattr(lib, entry)(dy.data_ptr(), kind, M, N, q.codes.data_ptr(), q.scales.data_ptr(), K,
                                 L.elem_type(out.dtype), out.data_ptr(), L.ptr(offsets),
                                 0 if offsets is None else offsets.numel() - 1, L.ptr(ws), nbytes, L.stream_of(out))
    if rc:
        L.check(rc, f"{entry[4:]}({M}x{N} by {K})")
    return out


def _grad_a(dy: Tensor, b: mxfp4_tensor, dtype: torch.dtype, offsets: Optional[Tensor] = None) -> Tensor:
    """dy [M, N] @ dequantize(b) [N, K] (b [E, N, K] by expert), [M, K]."""
    out = torch.empty(dy.shape[0], b.shape[-1], dtype=dtype, device=dy.device)
    return _grad("mxk_mxfp4_grad_a", dy, b, out, offsets)


def _grad_b(dy: Tensor, a: mxfp4_tensor, dtype: torch.dtype, offsets: Optional[Tensor] = None) -> Tensor:
    """dy [M, N].T @ dequantize(a) [M, K], [N, K] ([E, N, K] by expert)."""
    shape = (dy.shape[1], a.shape[-1])
    out = torch.empty(shape if offsets is None else (offsets.numel() - 1, *shape), dtype=dtype, device=dy.device)
    return _grad("mxk_mxfp4_grad_b", dy, a, out, offsets)


def _grad_bias(dy: Tensor, dtype: torch.dtype, offsets: Optional[Tensor] = None) -> Tensor:
    """Column sums of dy, per expert where offsets are given: the gradient of b
    against one column of ones.  Of a float64 bias too, which the product rounds
    to float32."""
    codes = torch.zeros(dy.shape[0], 16, dtype=torch.uint8, device=dy.device)
    codes[:, 0] = 2  # the code of 1.0
    ones = mxfp4_tensor(codes, torch.full((dy.shape[0], 1), 127, dtype=torch.uint8, device=dy.device),
                        (dy.shape[0], 1))
    return _grad_b(dy, ones, dtype if dtype in _FLOATS else torch.float32, offsets).squeeze(-1).to(dtype)


def _pack_weight(weight: Union[Tensor, mxfp4_tensor]) -> mxfp4_tensor:
    return weight if isinstance(weight, mxfp4_tensor) else mxfp4_quantize(weight)


class _MXFP4Linear(torch.autograd.Function):
    """mxfp4_linear over [M, K] rows; `packed` is the weight where it is held
    packed (weight is then None)."""

    @staticmethod
    def forward(ctx, x, weight, bias, packed):
        b = packed if packed is not None else mxfp4_quantize(weight)
        a = mxfp4_quantize(x)
        out = torch.empty(x.shape[0], b.shape[0], dtype=x.dtype, device=x.device)
        _product(a, b, x.shape[0], b.shape[0], _bias_f32(bias, (b.shape[0],)), out)
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        kept = ((b.codes, b.scales) if need_x else (None, None)) + ((a.codes, a.scales) if need_w else (None, None))
        ctx.save_for_backward(*kept)
        ctx.sizes = (a.shape, b.shape, x.dtype, None if weight is None else weight.dtype,
                     None if bias is None else bias.dtype)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        bc, bs, ac, as_ = ctx.saved_tensors
        a_shape, b_shape, x_dtype, w_dtype, bias_dtype = ctx.sizes
        dy = dy.contiguous()
        dx = _grad_a(dy, mxfp4_tensor._of(bc, bs, b_shape), x_dtype) if ctx.needs_input_grad[0] else None
        dw = _grad_b(dy, mxfp4_tensor._of(ac, as_, a_shape), w_dtype) if ctx.needs_input_grad[1] else None
        db = _grad_bias(dy, bias_dtype) if ctx.needs_input_grad[2] else None
        return dx, dw, db, None


def _no_tangents(name: str, *tensors) -> None:
    """Refuse dual tensors: the kernels read the values alone, and a result would lose its tangent."""
    if forward_ad._current_level >= 0 and any(isinstance(t, Tensor) and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise L.MXKError(f"{name} has no forward-mode derivative")


def _check_linear(name: str, x: Tensor, weight, dims: int) -> None:
    if x.dtype not in _FLOATS:
        raise TypeError(f"{name}: x is float32, float16 or bfloat16, got {x.dtype}")
    if not isinstance(weight, mxfp4_tensor) and weight.dtype not in _FLOATS:
        raise TypeError(f"{name}: the weight is an mxfp4_tensor or a float tensor, got {weight.dtype}")
    shape = weight.shape
    if len(shape) != dims or x.dim() < 1 or x.shape[-1] != shape[-1]:
        want = "[N, K]" if dims == 2 else "[E, N, K]"
        raise ValueError(f"{name}: x [..., K] and a weight {want} expected, got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")


def _wants_grad(x: Tensor, weight, bias: Optional[Tensor]) -> bool:
    return (x.requires_grad or bias is not None and bias.requires_grad
            or not isinstance(weight, mxfp4_tensor) and weight.requires_grad) and torch.is_grad_enabled()


def mxfp4_linear(x: Tensor, weight: Union[Tensor, mxfp4_tensor], bias: Optional[Tensor] = None) -> Tensor:
    """x [..., K] packed to 4 bits, times weight [N, K].T (+ bias [N]), as x's
    dtype.  weight: an mxfp4_tensor (held packed, no gradient) or a float
    tensor, packed in the call and differentiable."""
    _check_linear("mxfp4_linear", x, weight, 2)
    _no_tangents("mxfp4_linear", x, weight, bias)
    N, K = weight.shape
    x2 = x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), K)
    if _wants_grad(x, weight, bias):
        held = isinstance(weight, mxfp4_tensor)
        y = _MXFP4Linear.apply(x2, None if held else weight, bias, weight if held else None)
    else:
        y = _linear(x2, _pack_weight(weight), x2.shape[0], _bias_f32(bias, (N,)))
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], N)
