"""Serving from a paged 8-bit key-value cache: rotary positions, new tokens into
the pages, attention over them, and the accepted path of a drafted tree.

  rotary_table(freqs, axis)          how positions turn a head's pairs
  rotary(x, positions, table)        heads rotated; differentiable
  kv_batch(table, lengths, offsets)  the sequences of a step
  kv_pages(codes, scales)            the pool of pages (kv_pages.empty makes one)
    .append(k, v, batch, ...)        keys (and queries) rotated, keys and values packed
    .attend(q, batch, mask)          attention of the new tokens, causal or by a mask
    .keep(batch, path)               accepted drafted tokens moved behind the context
    .read(batch, tokens)             values of positions

``kv_cache_quantizer`` holds one batch's steps in a ring and gives them back
as float32; here sequences share a pool, and the attention reads the codes
as they lie.  No call waits for the GPU: lengths and pages stay on the
device, so that a step can be recorded in a graph and replayed with others.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import _lib as L
from .microscale import _FLOATS, _no_tangents
from .tensor import mx_tensor

Tensor = torch.Tensor

_HEADS = (64, 128, 256)
_MANY = 1 << 30  # more tokens than a batch has


def _together(first: Tensor, *rest: Optional[Tensor]) -> int:
    """The GPU that all tensors are on."""
    index = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != index:
            L.require_gpu(first, *rest)  # names the two
    if index < 0:
        L.require_gpu(first)
    return index


def _no_gradients(name: str, x: Tensor) -> None:
    """Refuse a tensor that would need a gradient or a tangent."""
    if x.requires_grad and torch.is_grad_enabled():
        raise L.MXKError(f"{name} has no gradient: call it under torch.no_grad(), or with detached tensors")
    _no_tangents(name, x)


def _values(name: str, x: Tensor) -> Tensor:
    """A packed tensor's values; a tensor that would need a gradient or a tangent is refused."""
    if isinstance(x, mx_tensor):
        x = x.dequantize()
    _no_gradients(name, x)
    return x


# ---------------------------------------------------------------- rotary positions
class rotary_table:
    """Angles of rotary positions: pair i of a head turns by ``freqs[i]`` radians
    for each position on axis ``axis[i]``.

    freqs float64 [pairs] and axis int32 [pairs] (None: one axis) on the GPU, used as
    they are: a change in place counts for the calls after it, and a gradient of a call
    before it is refused as torch refuses its own.  Pair i is elements (i, i + pairs), or
    (2i, 2i + 1) where ``interleaved``; a head's elements from 2 * pairs on are not rotated.
    Nothing is differentiable towards freqs: calls refuse them where they would need a gradient."""

    __slots__ = ("freqs", "axis", "interleaved")

    def __init__(self, freqs: Tensor, axis: Optional[Tensor] = None, *, interleaved: bool = False):
        if freqs.dtype != torch.float64 or freqs.dim() != 1:
            raise TypeError(f"rotary_table: freqs [pairs] in float64 expected, got {tuple(freqs.shape)} in {freqs.dtype}")
        if axis is not None and (axis.dtype != torch.int32 or axis.shape != freqs.shape):
            raise TypeError(f"rotary_table: axis [pairs] in int32 expected, got {tuple(axis.shape)} in {axis.dtype}")
        L.require_gpu(freqs, axis)
        self.freqs = freqs.contiguous()
        self.axis = None if axis is None else axis.contiguous()
        self.interleaved = bool(interleaved)

    @classmethod
    def make(cls, rotated: int, base: float = 10000.0, *, sections: Optional[Sequence[int]] = None,
             restart: bool = False, interleaved: bool = False, device="cuda") -> "rotary_table":
        """The table of frequencies base ** (-i / pairs) for the pairs i of `rotated` elements.

        sections: how many pairs each axis has, one after the other (time,
        height, width); restart begins each axis' frequencies anew, as for
        images whose axes are alike."""
        if rotated < 0 or rotated % 2:
            raise ValueError(f"rotary_table: an even number of rotated elements expected, got {rotated}")
        pairs = rotated // 2
        if sections is not None and (sum(sections) != pairs or any(s < 0 for s in sections)):
            raise ValueError(f"rotary_table: sections that add up to {pairs} pairs expected, got {tuple(sections)}")
        parts = [pairs] if sections is None else list(sections)
        spans = parts if restart else [pairs] * len(parts)
        freqs, axis, first = [], [], 0
        for a, (n, span) in enumerate(zip(parts, spans)):
            freqs += [float(base) ** (-(i if restart else first + i) / span) for i in range(n)]
            axis += [a] * n
            first += n
        return cls(torch.tensor(freqs, dtype=torch.float64, device=device),
                   None if sections is None else torch.tensor(axis, dtype=torch.int32, device=device),
                   interleaved=interleaved)

    def __repr__(self):
        return f"rotary_table(pairs={self.freqs.numel()}, interleaved={self.interleaved})"


def _positions(name: str, positions: Tensor, lead) -> Tuple[Tensor, int]:
    """Contiguous positions and their number of axes; lead: the shape of the tokens."""
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: positions are int32 or int64, got {positions.dtype}")
    shape = positions.shape
    if shape == lead:
        axes = 1
    elif len(shape) == len(lead) + 1 and shape[:-1] == lead and shape[-1] > 0:
        axes = shape[-1]
    else:
        raise ValueError(f"{name}: positions {tuple(lead)}, or with their axes last, expected, got "
                         f"{tuple(positions.shape)}")
    return positions.contiguous(), axes


def _token_rows(x: Tensor) -> Tensor:
    """x [..., H, D] as [tokens, H, D] with D contiguous, without a copy where its strides allow."""
    if x.dim() != 3:
        x = x.reshape(math.prod(x.shape[:-2]), *x.shape[-2:])
    return x if x.stride(2) == 1 or x.shape[2] <= 1 else x.contiguous()


def _rotary(x: Tensor, positions: Tensor, axes: int, freqs: Tensor, axis: Optional[Tensor], interleaved: bool,
            backward: bool) -> Tensor:
    gpu = _together(x, positions, freqs, axis)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    rows = _token_rows(x)
    tokens, H, D = rows.shape
    token, head, _ = rows.stride()
    with L.on_gpu(gpu):
        rc = L.lib().mxk_rotary(rows.data_ptr(), _FLOATS[x.dtype], tokens, H, D, token, head, freqs.data_ptr(),
                                L.ptr(axis), freqs.numel(), interleaved, positions.data_ptr(),
                                positions.element_size(), axes, backward, y.data_ptr(), L.stream_on(gpu))
    if rc:
        L.check(rc, f"rotary({tokens}x{H}x{D})")
    return y


class _Rotary(torch.autograd.Function):
    """Linear in x: its gradient is the opposite rotation, to any order."""

    @staticmethod
    def forward(ctx, x, positions, axes, freqs, axis, interleaved, backward):
        ctx.save_for_backward(positions, freqs, axis)
        ctx.how = axes, interleaved, backward
        return _rotary(x, positions, axes, freqs, axis, interleaved, backward)

    @staticmethod
    def backward(ctx, dy):
        positions, freqs, axis = ctx.saved_tensors
        axes, interleaved, backward = ctx.how
        turn = _Rotary.apply if torch.is_grad_enabled() and dy.requires_grad else _rotary
        return turn(dy, positions, axes, freqs, axis, interleaved, not backward), None, None, None, None, None, None


def rotary(x: Tensor, positions: Tensor, table: rotary_table) -> Tensor:
    """Heads x [..., heads, D] (float32, float16 or bfloat16, any strides)
    rotated by their tokens' positions [...] or [..., axes] (int32 or int64; an
    axis of the table that they lack is at position 0).

    Angles are reduced in float64, so that far positions keep them; products
    and sums are float32, rounded once.  The gradient is the opposite rotation
    of the output's, itself differentiable.  Positions without axes, or with one,
    are the same for all pairs."""
    if isinstance(x, mx_tensor):
        x = x.dequantize()
    if x.dtype not in _FLOATS:
        raise TypeError(f"rotary: float32, float16 or bfloat16 expected, got {x.dtype}")
    if x.dim() < 2:
        raise ValueError(f"rotary: [..., heads, D] expected, got {tuple(x.shape)}")
    _no_tangents("rotary", x)
    positions, axes = _positions("rotary", positions, x.shape[:-2])
    if 2 * table.freqs.numel() > x.shape[-1]:
        raise ValueError(f"rotary: the table rotates {2 * table.freqs.numel()} elements, a head has {x.shape[-1]}")
    _no_gradients("rotary towards a table's frequencies", table.freqs)
    turn = _Rotary.apply if x.requires_grad and torch.is_grad_enabled() else _rotary
    return turn(x, positions, axes, table.freqs, table.axis, table.interleaved, False)


# ---------------------------------------------------------------- the paged cache
class kv_batch(NamedTuple):
    """The sequences of one step, int32 tensors on the GPU.

    table    [B, width]  page of each run of page_size positions; entries that
                         a sequence does not use may be anything outside the pool (-1)
    lengths  [B]         positions each sequence holds before the step
    offsets  [B + 1]     ascending: sequence b's new tokens are rows offsets[b] to
                         offsets[b + 1] of the step's tensors (none for an idle one)

    New token i of sequence b has position lengths[b] + i.  Rows in front of
    offsets[0] and from offsets[B] on are padding: nothing is stored for them,
    and results have zeros there."""
    table: Tensor
    lengths: Tensor
    offsets: Tensor


def kv_tree_mask(parents: Sequence[int], device="cuda") -> Tuple[Tensor, Tensor]:
    """Mask words int64 [n, words] and depths int32 [n] of a tree of drafted
    tokens: parents[i] < i, or negative for a root.  A token sees itself and the
    tokens on its way from the root.  Host data to device tensors: made once for a
    tree, repeated for the sequences that draft with it."""
    seen, depth = [], []
    for i, p in enumerate(parents):
        p = int(p)
        if p >= i:
            raise ValueError(f"kv_tree_mask: token {i} comes before its parent {p}")
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    words = max(1, -(-len(seen) // 64))
    full = (1 << 64) - 1
    rows = [[(m >> 64 * w & full) - (1 << 64 if m >> 64 * w + 63 & 1 else 0) for w in range(words)] for m in seen]
    return (torch.tensor(rows, dtype=torch.int64, device=device).view(-1, words),
            torch.tensor(depth, dtype=torch.int32, device=device))


def _check_batch(name: str, batch: kv_batch) -> None:
    table, lengths, offsets = batch
    if not (table.dtype == lengths.dtype == offsets.dtype == torch.int32
            and table.is_contiguous() and lengths.is_contiguous() and offsets.is_contiguous()):
        raise TypeError(f"{name}: a batch's tensors are contiguous int32, got {table.dtype}, {lengths.dtype} and "
                        f"{offsets.dtype}")
    shape = table.shape
    if len(shape) != 2 or lengths.shape != shape[:1] or offsets.shape != (shape[0] + 1,):
        raise ValueError(f"{name}: a batch has table [B, width], lengths [B] and offsets [B + 1], got "
                         f"{tuple(table.shape)}, {tuple(lengths.shape)} and {tuple(offsets.shape)}")


class kv_pages:
    """A pool of pages of 8-bit keys and values: ``codes`` int8 [pages, 2, heads,
    page_size, head_dim] (keys, then values) and ``scales`` float32 [pages, 2,
    heads, page_size], value = code * scale, as kv_cache_quantizer's "int8dv".

    page_size is a power of two from 16 on, head_dim 64, 128 or 256.  Which
    sequence has which page is the caller's: pages are named by a kv_batch alone.
    A page may stand in several tables (a shared prefix) while nobody writes to it.
    Scales that require a gradient are refused by the calls where gradients are recorded."""

    __slots__ = ("codes", "scales")

    def __init__(self, codes: Tensor, scales: Tensor):
        if codes.dtype != torch.int8 or scales.dtype != torch.float32:
            raise TypeError(f"kv_pages: int8 codes and float32 scales expected, got {codes.dtype} and {scales.dtype}")
        shape = codes.shape
        if len(shape) != 5 or shape[1] != 2 or scales.shape != shape[:-1]:
            raise ValueError(f"kv_pages: codes [pages, 2, heads, page_size, head_dim] and scales [pages, 2, heads, "
                             f"page_size] expected, got {tuple(shape)} and {tuple(scales.shape)}")
        if shape[2] < 1 or shape[3] < 16 or shape[3] & (shape[3] - 1) or shape[4] not in _HEADS:
            raise ValueError(f"kv_pages: one head at least, a page of a power of two of positions from 16 on and heads "
                             f"of 64, 128 or 256 expected, got {tuple(shape)}")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("kv_pages: codes and scales are written in place: contiguous tensors expected")
        L.require_gpu(codes, scales)
        if codes.data_ptr() % 16 or scales.data_ptr() % 16:
            raise ValueError("kv_pages: codes and scales start on 16 bytes")
        self.codes, self.scales = codes, scales

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_heads: int, head_dim: int, device="cuda") -> "kv_pages":
        """A pool of its own.  Positions that nothing was stored for read as zeros: a step that is run or recorded
        ahead of its tokens attends what the pool defines, not what its memory held before."""
        return cls(torch.empty(n_pages, 2, n_heads, page_size, head_dim, dtype=torch.int8, device=device),
                   torch.zeros(n_pages, 2, n_heads, page_size, dtype=torch.float32, device=device))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()

    def _pool(self, name: str):
        """Addresses and sizes for a call; scales that need a gradient or a tangent are refused as its tensors are."""
        _no_gradients(name, self.scales)
        n, _, H, page, D = self.codes.shape
        return self.codes.data_ptr(), self.scales.data_ptr(), n, page, H, D

    def _written(self) -> None:
        """The pool's tensors count as changed in place, for what autograd has saved of them."""
        torch.autograd.graph.increment_version((self.codes, self.scales))

    def _rows(self, name: str, what: str, x: Tensor, H: int, D: int) -> Tensor:
        """x [tokens, heads, D] with D contiguous; H: heads of keys and values, whose multiple queries have."""
        x = _values(name, x)
        shape = x.shape
        if len(shape) != 3 or shape[2] != D or (what != "q" and shape[1] != H):
            raise ValueError(f"{name}: {what} [tokens, {'heads' if what == 'q' else H}, {D}] expected, got {tuple(shape)}")
        if what == "q" and (shape[1] < H or shape[1] % H):
            raise ValueError(f"{name}: query heads in groups of one size for each of {H} heads expected, got {shape[1]}")
        return x if x.stride(2) == 1 else x.contiguous()

    def append(self, k: Tensor, v: Tensor, batch: kv_batch, *, rotary: Optional[rotary_table] = None,
               positions: Optional[Tensor] = None, q: Optional[Tensor] = None) -> Optional[Tensor]:
        """Store the new tokens' keys and values k, v [tokens, heads, head_dim]
        (float32, float16 or bfloat16, heads contiguous) at their positions.

        With a rotary table keys are rotated on the way, by positions [tokens] or
        [tokens, axes] (None: each token's position in its sequence, on every
        axis); they are packed from the unrounded float32 rotation.  q [tokens, q_heads,
        head_dim] is rotated along and returned.  A head's row with a NaN or an
        infinity reads as NaN.  Nothing is differentiable: tensors that require a
        gradient are refused where gradients are recorded."""
        codes, scales, n, page, H, D = self._pool("kv_pages.append")
        k, v = self._rows("kv_pages.append", "k", k, H, D), self._rows("kv_pages.append", "v", v, H, D)
        if q is not None:
            q = self._rows("kv_pages.append", "q", q, H, D)
        kind = _FLOATS.get(k.dtype)
        if kind is None or v.dtype != k.dtype or q is not None and q.dtype != k.dtype:
            raise TypeError(f"kv_pages.append: keys, values and queries of one type (float32, float16 or bfloat16) "
                            f"expected, got {k.dtype}, {v.dtype}{'' if q is None else f' and {q.dtype}'}")
        T = k.shape[0]
        if v.shape[0] != T or q is not None and q.shape[0] != T:
            raise ValueError(f"kv_pages.append: one row for each of {T} tokens expected, got {v.shape[0]} of v"
                             f"{'' if q is None else f' and {q.shape[0]} of q'}")
        _check_batch("kv_pages.append", batch)
        table, lengths, offsets = batch
        freqs = axis = None
        pairs = axes = bytes_ = interleaved = 0
        if rotary is not None:
            freqs, axis, interleaved = rotary.freqs, rotary.axis, rotary.interleaved
            _no_gradients("kv_pages.append towards a table's frequencies", freqs)
            pairs = freqs.numel()
            if 2 * pairs > D:
                raise ValueError(f"kv_pages.append: the table rotates {2 * pairs} elements, a head has {D}")
            if positions is not None:
                positions, axes = _positions("kv_pages.append", positions, (T,))
                bytes_ = positions.element_size()
        elif positions is not None or q is not None:
            raise ValueError("kv_pages.append: positions and queries go with a rotary table")
        gpu = _together(self.codes, k, v, q, positions, freqs, axis, table, lengths, offsets)
        out, qt, qh, Hq = None, 0, 0, 0
        if q is not None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            (qt, qh, _), Hq = q.stride(), q.shape[1]
        (kt, kh, _), (vt, vh, _), (B, width) = k.stride(), v.stride(), table.shape
        with L.on_gpu(gpu):
            rc = L.lib().mxk_kv_pages_append(
                k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, L.ptr(q), qt, qh, Hq, kind, codes, scales, n, page, H, D,
                table.data_ptr(), lengths.data_ptr(), offsets.data_ptr(), B, width, T, L.ptr(freqs), L.ptr(axis), pairs,
                interleaved, L.ptr(positions), bytes_, axes, L.ptr(out), L.stream_on(gpu))
        if rc:
            L.check(rc, f"kv_pages.append({T} tokens, {H} heads of {D})")
        self._written()
        return out

    def attend(self, q: Tensor, batch: kv_batch, *, mask: Optional[Tensor] = None,
               scale: Optional[float] = None) -> Tensor:
        """Attention of the new tokens' queries q [tokens, q_heads, head_dim]
        over the pages of their sequences, whose new keys and values are stored
        already (append).  q_heads is a multiple of the pool's heads: query
        head i reads head i // (q_heads // heads).

        A token sees all positions its sequence held before the step, and of
        the step's own tokens those up to itself; with mask (int64 [tokens,
        words]) those, in any order, whose bit is set: bit j % 64 of word j // 64
        is new token j of the same sequence.  scale: of the scores, 1 /
        sqrt(head_dim) unless given.  A row that sees nothing is zeros.

        Codes are used as they are and sums are float32.  Where a sequence has
        few rows a head (64 on average; 96 in float32 and with heads of 256), q keeps 16
        bits of its row's largest element (24 in float32), and a probability times
        its value's scale 11 bits (22 in float32 and float16) down to 2^-24 of
        the largest that the row sees.  Else q's elements keep 11 bits (22 in float32) down to 2^-20 of
        their row's largest, and those products 11 (22 in float32) down to 2^-20, in bfloat16 with two
        roundings more and down to 2^-10.  Nothing is differentiable, as in append."""
        codes, scales, n, page, H, D = self._pool("kv_pages.attend")
        q = self._rows("kv_pages.attend", "q", q, H, D)
        kind = _FLOATS.get(q.dtype)
        if kind is None:
            raise TypeError(f"kv_pages.attend: float32, float16 or bfloat16 expected, got {q.dtype}")
        _check_batch("kv_pages.attend", batch)
        T, Hq, _ = q.shape
        words = 0
        if mask is not None:
            if mask.dtype != torch.int64:
                raise TypeError(f"kv_pages.attend: a mask of int64 words expected, got {mask.dtype}")
            if mask.dim() != 2 or mask.shape[0] != T or mask.shape[1] < 1:
                raise ValueError(f"kv_pages.attend: a mask [{T}, words] expected, got {tuple(mask.shape)}")
            mask = mask.contiguous()
            words = mask.shape[1]
        scale = D ** -0.5 if scale is None else float(scale)
        if not (scale > 0.0 and math.isfinite(scale)):
            raise ValueError(f"kv_pages.attend: a positive scale expected, got {scale}")
        table, lengths, offsets = batch
        gpu = _together(self.codes, q, mask, table, lengths, offsets)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lib = L.lib()
        (qt, qh, _), (B, width) = q.stride(), table.shape
        nbytes = lib.mxk_kv_pages_attend_workspace(kind, T, B, width, page, H, Hq, D)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        with L.on_gpu(gpu):
            rc = lib.mxk_kv_pages_attend(q.data_ptr(), kind, qt, qh, Hq, codes, scales, n, page, H, D, table.data_ptr(),
                                         lengths.data_ptr(), offsets.data_ptr(), B, width, T, L.ptr(mask), words, scale,
                                         out.data_ptr(), L.ptr(ws), nbytes, L.stream_on(gpu))
        if rc:
            L.check(rc, f"kv_pages.attend({T} tokens, {Hq} heads of {D})")
        return out

    def keep(self, batch: kv_batch, path: Tensor) -> None:
        """Move the accepted tokens of a step behind the context: position
        lengths[b] + j takes the keys and values of the step's token path[b, j]
        (int32 [B, steps], at most 64 steps; an entry outside the sequence's new
        tokens, as -1, moves nothing).  All are read before any is written.  The
        caller then adds the number accepted to lengths."""
        _check_batch("kv_pages.keep", batch)
        table, lengths, offsets = batch
        if path.dtype != torch.int32:
            raise TypeError(f"kv_pages.keep: a path of int32 expected, got {path.dtype}")
        if path.dim() != 2 or path.shape[0] != table.shape[0]:
            raise ValueError(f"kv_pages.keep: a path [{table.shape[0]}, steps] expected, got {tuple(path.shape)}")
        path = path.contiguous()
        gpu = _together(self.codes, path, table, lengths, offsets)
        codes, scales, n, page, H, D = self._pool("kv_pages.keep")
        with L.on_gpu(gpu):
            rc = L.lib().mxk_kv_pages_keep(codes, scales, n, page, H, D, table.data_ptr(), lengths.data_ptr(),
                                           offsets.data_ptr(), table.shape[0], table.shape[1], _MANY, path.data_ptr(),
                                           path.shape[1], L.stream_on(gpu))
        if rc:
            L.check(rc, f"kv_pages.keep({tuple(path.shape)})")
        self._written()

    def read(self, batch: kv_batch, tokens: int, dtype: torch.dtype = torch.bfloat16) -> Tuple[Tensor, Tensor]:
        """Keys and values [tokens, heads, head_dim] at positions lengths[b] + i,
        row offsets[b] + i; zeros where there is none.  (A sequence's whole history:
        lengths of 0 and offsets that count it.)  tokens: rows of the result."""
        _check_batch("kv_pages.read", batch)
        if tokens < 0:
            raise ValueError(f"kv_pages.read: a number of tokens expected, got {tokens}")
        kind = L.elem_type(dtype)
        table, lengths, offsets = batch
        gpu = _together(self.codes, table, lengths, offsets)
        codes, scales, n, page, H, D = self._pool("kv_pages.read")
        k = torch.empty((tokens, H, D), dtype=dtype, device=self.codes.device)
        v = torch.empty_like(k)
        with L.on_gpu(gpu):
            rc = L.lib().mxk_kv_pages_read(codes, scales, n, page, H, D, table.data_ptr(), lengths.data_ptr(),
                                           offsets.data_ptr(), table.shape[0], table.shape[1], tokens, kind,
                                           k.data_ptr(), v.data_ptr(), L.stream_on(gpu))
        if rc:
            L.check(rc, f"kv_pages.read({tokens} tokens)")
        return k, v

    def __repr__(self):
        n, _, H, page, D = self.codes.shape
        return f"kv_pages(pages={n}, page_size={page}, heads={H}, head_dim={D}, device={self.device})"
