"""Layers of experts on packed weights: tokens sorted by expert, each
segment through its expert's microscaled 4-bit weight, and the rows of a token
weighted and added.

  expert_sort(ids, n_experts)                 -> expert_plan
  expert_gather(x, plan)                      token rows in the plan's order
  expert_linear(x, weight, plan, bias)        rows through their expert's weight
  expert_combine(h, plan, gates)              rows back to tokens
  mxfp4_expert_mlp                            the layer built from them

No call waits for the GPU: segment lengths stay on the device.  Every sum has a
fixed order, so results do not change from run to run.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib as L
from .microscale import (_FLOATS, _bias_f32, _check_linear, _grad_a, _grad_b, _grad_bias, _linear, _no_tangents,
                         _pack_weight, _product, _row_major, _wants_grad, mxfp4_quantize, mxfp4_tensor)

Tensor = torch.Tensor


class expert_plan(NamedTuple):
    """Order of the picks of a routing [tokens, top] by expert, int32 arrays.

    order    [tokens * top]  the pick (token * top + j) at each place, stable;
                             -1 past the last pick that has an expert
    place    [tokens, top]   the place of each pick; -1 for a pick without an
                             expert here (its id is outside [0, n_experts))
    offsets  [n_experts + 1] first place of each expert's rows; the last entry
                             is the number of places in use

    A pick may be dropped after the sort (an expert over its capacity) by a
    place of -1: expert_combine follows the places alone and passes the pick's
    row a gradient of zero.  expert_gather and expert_linear follow order, so that
    the row is still computed unless its order is -1 too; a row without a place passes
    a gathered x no gradient.

    Some experts' part of a plan (those of this device) is the plan with
    offsets[first : first + number + 1]: expert_linear computes their rows and
    leaves zeros in all others, in front of them and behind.
    """
    order: Tensor
    place: Tensor
    offsets: Tensor


def expert_sort(ids: Tensor, n_experts: int) -> expert_plan:
    """The plan of expert ids [tokens, top] (int32 or int64); at most 1000
    experts.  An id outside [0, n_experts) has no expert here (a padded
    token, or an expert of another device)."""
    if ids.dim() != 2 or ids.shape[1] < 1:
        raise ValueError(f"expert_sort: ids [tokens, top] with top >= 1 expected, got {tuple(ids.shape)}")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"expert_sort: ids are int32 or int64, got {ids.dtype}")
    dev = L.require_gpu(ids)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    P = ids.numel()
    place = torch.empty_like(ids, dtype=torch.int32)
    order = torch.empty((P,), dtype=torch.int32, device=dev)
    offsets = torch.empty((max(n_experts, 0) + 1,), dtype=torch.int32, device=dev)
    lib = L.lib()
    nbytes = lib.mxk_expert_sort_workspace(P, n_experts)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with L.on_device(dev):
        rc = lib.mxk_expert_sort(ids.data_ptr(), ids.element_size(), P, n_experts, order.data_ptr(), place.data_ptr(),
                                 offsets.data_ptr(), L.ptr(ws), nbytes, L.stream_of(ids))
    if rc:
        L.check(rc, f"expert_sort({P} picks, {n_experts} experts)")
    return expert_plan(order, place, offsets)


def _check_plan(name: str, plan: expert_plan) -> None:
    order, place, offsets = plan
    if not (order.dtype == place.dtype == offsets.dtype == torch.int32
            and order.is_contiguous() and place.is_contiguous() and offsets.is_contiguous()):
        raise TypeError(f"{name}: a plan's tensors are contiguous int32, got "
                        f"{order.dtype}, {place.dtype} and {offsets.dtype}")
    if order.dim() != 1 or place.dim() != 2 or place.numel() != order.numel() or offsets.dim() != 1 \
            or offsets.numel() < 2:
        raise ValueError(f"{name}: a plan has order [tokens * top], place [tokens, top] and offsets [experts + 1], got "
                         f"{tuple(order.shape)}, {tuple(place.shape)} and {tuple(offsets.shape)}")


def _float_rows(name: str, x: Tensor, rows: int, what: str) -> None:
    if x.dtype not in _FLOATS:
        raise TypeError(f"{name}: float32, float16 or bfloat16 expected, got {x.dtype}")
    if x.dim() != 2 or x.shape[0] != rows:
        raise ValueError(f"{name}: [{rows}, columns] ({what}) expected, got {tuple(x.shape)}")


def _gather(x: Tensor, plan: expert_plan) -> Tensor:
    order = plan.order
    dev = L.require_gpu(x, order)
    x = _row_major(x)
    tokens, top = plan.place.shape
    cols = x.shape[1]
    out = torch.empty((tokens * top, cols), dtype=x.dtype, device=dev)
    with L.on_device(dev):
        rc = L.lib().mxk_expert_gather(x.data_ptr(), x.element_size(), tokens, cols, x.stride(0), order.data_ptr(),
                                       tokens * top, top, out.data_ptr(), L.stream_of(out))
    if rc:
        L.check(rc, f"expert_gather({tokens}x{cols}, top {top})")
    return out


def _combine(h: Tensor, plan: expert_plan, gates: Optional[Tensor], dtype: Optional[torch.dtype] = None) -> Tensor:
    place, dtype = plan.place, dtype or h.dtype
    dev = L.require_gpu(h, gates, place)
    h = h.contiguous()
    tokens, top = place.shape
    rows, cols = h.shape
    y = torch.empty((tokens, cols), dtype=dtype, device=dev)
    with L.on_device(dev):
        rc = L.lib().mxk_expert_combine(h.data_ptr(), _FLOATS[h.dtype], rows, place.data_ptr(), L.ptr(gates), tokens,
                                        top, cols, _FLOATS[dtype], y.data_ptr(), L.stream_of(y))
    if rc:
        L.check(rc, f"expert_combine({tokens}x{cols}, top {top})")
    return y


class _ExpertGather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.save_for_backward(*plan)
        return _gather(x, plan)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return _combine(dy, expert_plan(*ctx.saved_tensors), None), None


class _ExpertCombine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, gates, plan):
        h = h.contiguous()
        ctx.save_for_backward(None if gates is None else h, gates, *plan)
        return _combine(h, plan, gates)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        h, gates, *plan = ctx.saved_tensors
        plan = expert_plan(*plan)
        dy = dy.contiguous()
        dev = L.require_gpu(dy, h, gates, *plan)
        tokens, top = plan.place.shape
        rows, cols = tokens * top, dy.shape[1]
        dh = torch.empty((rows, cols), dtype=dy.dtype, device=dev)
        dg = None if gates is None else torch.empty_like(gates)
        with L.on_device(dev):
            rc = L.lib().mxk_expert_combine_grad(dy.data_ptr(), L.ptr(h), L.elem_type(dy.dtype), rows,
                                                 plan.order.data_ptr(), plan.place.data_ptr(), L.ptr(gates), tokens,
                                                 top, cols, dh.data_ptr(), L.ptr(dg), L.stream_of(dy))
        if rc:
            L.check(rc, f"expert_combine gradient({tokens}x{cols}, top {top})")
        return dh, dg, None


def expert_gather(x: Tensor, plan: expert_plan) -> Tensor:
    """Rows of x [tokens, D] in the plan's order, [tokens * top, D]: row r is
    x[order[r] // top], zeros past the places in use.  The gradient of a token is
    the sum of its rows' (in float32, by ascending pick)."""
    _check_plan("expert_gather", plan)
    _float_rows("expert_gather", x, plan.place.shape[0], "one row per token")
    _no_tangents("expert_gather", x)
    if x.requires_grad and torch.is_grad_enabled():
        return _ExpertGather.apply(x, plan)
    return _gather(x, plan)


def expert_combine(h: Tensor, plan: expert_plan, gates: Optional[Tensor] = None) -> Tensor:
    """Sum over each token's picks of gates[t, j] * h[place[t, j]], [tokens, D],
    added in float32 by ascending j and rounded once; a pick without a place
    adds nothing, and a row that no place names has a gradient of zero (one
    place at most names a row).  gates [tokens, top] (float; None: ones).  Differentiable
    in h and gates."""
    _check_plan("expert_combine", plan)
    _float_rows("expert_combine", h, plan.order.numel(), "one row per pick")
    _no_tangents("expert_combine", h, gates)
    if gates is not None:
        if gates.shape != plan.place.shape:
            raise ValueError(f"expert_combine: gates {tuple(plan.place.shape)} expected, got {tuple(gates.shape)}")
        if gates.is_complex():
            raise TypeError(f"expert_combine: real gates expected, got {gates.dtype}")
        gates = gates.float().contiguous()
    if (h.requires_grad or gates is not None and gates.requires_grad) and torch.is_grad_enabled():
        return _ExpertCombine.apply(h, gates, plan)
    return _combine(h, plan, gates)


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, packed, plan, gather):
        b = packed if packed is not None else mxfp4_quantize(weight)
        a = mxfp4_quantize(x)
        y = _expert_product(a, b, plan, bias, gather, x.dtype)
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        kept = (b.codes, b.scales) if need_x else (None, None)
        # with gather the weight's gradient needs the rows in order: they are fetched in the backward pass
        kept += ((x, None) if gather else (a.codes, a.scales)) if need_w else (None, None)
        ctx.save_for_backward(*kept, *plan)
        ctx.sizes = (a.shape, b.shape, x.dtype, None if weight is None else weight.dtype,
                     None if bias is None else bias.dtype, gather)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        bc, bs, ac, as_, *plan = ctx.saved_tensors
        plan = expert_plan(*plan)
        a_shape, b_shape, x_dtype, w_dtype, bias_dtype, gather = ctx.sizes
        dy = dy.contiguous()
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            # a token's rows are added in float32, where parts beyond float16's range may cancel
            dx = _grad_a(dy, mxfp4_tensor._of(bc, bs, b_shape), torch.float32 if gather else x_dtype, plan.offsets)
            if gather:
                dx = _combine(dx, plan, None, x_dtype)
        if ctx.needs_input_grad[1]:
            a = mxfp4_quantize(_gather(ac, plan)) if gather else mxfp4_tensor._of(ac, as_, a_shape)
            dw = _grad_b(dy, a, w_dtype, plan.offsets)
        if ctx.needs_input_grad[2]:
            db = _grad_bias(dy, bias_dtype, plan.offsets)
        return dx, dw, db, None, None, None


def _expert_product(a: mxfp4_tensor, b: mxfp4_tensor, plan: expert_plan, bias: Optional[Tensor], gather: bool,
                    dtype: torch.dtype) -> Tensor:
    E, N, _ = b.shape
    rows = plan.order.numel()
    y = torch.empty(rows, N, dtype=dtype, device=a.device)
    return _product(a, b, rows, N, _bias_f32(bias, (E, N)), y, plan.offsets, plan.order if gather else None,
                    plan.place.shape[1])


def expert_linear(x: Tensor, weight: Union[Tensor, mxfp4_tensor], plan: expert_plan, bias: Optional[Tensor] = None,
                  *, gather: bool = False) -> Tensor:
    """Each expert's rows through its weight: y[r] = x[r] @ weight[e].T (+
    bias[e]) for the rows r of expert e, zeros in rows that no expert has.

    x [tokens * top, K] in the plan's order, packed to 4 bits in the call; with
    gather x is [tokens, K] and row r reads token order[r] // top, so that a
    token is packed once and not copied.  weight [E, N, K]: an mxfp4_tensor, or
    a float tensor, packed in the call and differentiable.  Returns
    [tokens * top, N] of x's dtype; gradients as for mxfp4_linear."""
    _check_linear("expert_linear", x, weight, 3)
    _no_tangents("expert_linear", x, weight, bias)
    _check_plan("expert_linear", plan)
    tokens, top = plan.place.shape
    _float_rows("expert_linear", x, tokens if gather else tokens * top,
                "one row per token" if gather else "one row per pick")
    if weight.shape[0] != plan.offsets.numel() - 1:
        raise ValueError(f"expert_linear: the plan has {plan.offsets.numel() - 1} experts, the weight {weight.shape[0]}")
    if _wants_grad(x, weight, bias):
        held = isinstance(weight, mxfp4_tensor)
        return _ExpertLinear.apply(x, None if held else weight, bias, weight if held else None, plan, gather)
    b = _pack_weight(weight)
    return _linear(x, b, tokens * top, _bias_f32(bias, tuple(b.shape[:2])), plan.offsets,
                   plan.order if gather else None, top)


class mxfp4_expert_mlp(nn.Module):
    """A feed-forward layer of experts on packed weights: the router picks
    `top` experts per token, each expert is SiLU(x @ gate.T) * (x @ up.T) @
    down.T, and the results are added with the softmax of the picked logits.

    router [E, D] stays float; up_gate [E, 2F, D] (gate rows first) and down
    [E, D, F] are packed once.  Inputs' and the router's gradients flow; packed
    weights have none."""

    def __init__(self, router: Tensor, up_gate: Tensor, down: Tensor, top: int):
        super().__init__()
        E, F2, D = up_gate.shape
        if router.shape != (E, D) or down.shape != (E, D, F2 // 2) or F2 % 2:
            raise ValueError(f"mxfp4_expert_mlp: router [E, D], up_gate [E, 2F, D] and down [E, D, F] expected, got "
                             f"{tuple(router.shape)}, {tuple(up_gate.shape)} and {tuple(down.shape)}")
        if not 1 <= top <= E:
            raise ValueError(f"mxfp4_expert_mlp: top from 1 to {E} expected, got {top}")
        self.top, self.sizes = top, (E, D, F2 // 2)
        self.router = nn.Parameter(router)
        for name, w in (("up_gate", up_gate), ("down", down)):
            q = mxfp4_quantize(w)
            self.register_buffer(name + "_codes", q.codes)
            self.register_buffer(name + "_scales", q.scales)

    def forward(self, x: Tensor) -> Tensor:
        E, D, F = self.sizes
        up_gate = mxfp4_tensor(self.up_gate_codes, self.up_gate_scales, (E, 2 * F, D))
        down = mxfp4_tensor(self.down_codes, self.down_scales, (E, D, F))
        rows = x.reshape(-1, D)
        logits, ids = nn.functional.linear(rows.float(), self.router.float()).topk(self.top, dim=1)
        plan = expert_sort(ids, E)
        h = expert_linear(rows, up_gate, plan, gather=True)
        h = nn.functional.silu(h[:, :F]) * h[:, F:]
        y = expert_combine(expert_linear(h, down, plan), plan, logits.softmax(1))
        return y.reshape(x.shape)

    def extra_repr(self):
        E, D, F = self.sizes
        return f"experts={E}, top={self.top}, d={D}, f={F}"
