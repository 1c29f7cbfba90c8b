"""Tokens by expert and back, and the experts' products on 4-bit weights, over torch tensors.

    sort(ids, experts, align=1)                       slots in the order of their experts -> Routing
    gather(x, routing)                                the tokens' rows in that order
    combine(z, routing, weights=None)                 and back: y[t] = sum_j weights[t, j] z[row of slot (t, j)]
    combine_grad(dy, z, routing, weights=None)        the gradients of combine: (dz, dweights)
    matmul(x, w, ids, weights)                        y[t] = sum_j weights[t, j] W[ids[t, j]] x[t], all of the above and mx4's product
    matmul_grad(dy, x, z, wt, routing, weights)       its gradients: (dx, dweights, dw)

The gradient of gather is combine without weights. What each computes, index by index, is in include/ozb.h (ozb_expert_*). Every call
is asynchronous on the current stream of the operands' device and may be captured into a CUDA graph; mx4.status() tells whether the
products of the last two did all that they were asked for. None takes part in autograd; they warn where an operand requires a gradient.
"""
from typing import NamedTuple

import torch

from ._lib import lib as _lib
from .mx4 import _MOST, _call, _codes, _cut, _offsets, _pitch, _result, _routed, _type

__all__ = ["Routing", "sort", "gather", "combine", "combine_grad", "matmul", "matmul_grad"]


class Routing(NamedTuple):
    """Where the slots (t, j) of T tokens go: expert e has the rows offsets[e] .. offsets[e + 1] - 1; rows [T, top] is the row of a slot
    (-1: dropped), slots [R] the slot t * top + j of a row (-1: none). All int32. align: what the segments are padded to (0: unknown)."""
    offsets: torch.Tensor
    rows: torch.Tensor
    slots: torch.Tensor
    align: int = 0


def _weights(weights, shape, index):
    if weights is None:
        return None
    if weights.dtype is not torch.float32 or weights.shape != shape or not weights.is_contiguous() or weights.get_device() != index:
        raise ValueError(f"weights must be contiguous float32 {tuple(shape)} on cuda:{index}")
    return weights.data_ptr()


def sort(ids, experts, align=1):
    """ids [T, top] (int32 or int64) -> Routing over `experts` experts, stable, segments padded to multiples of `align` (1 to 256; products
    along the tokens need 64). A number outside 0 .. experts - 1 drops its slot."""
    if ids.dtype not in (torch.int32, torch.int64) or ids.dim() != 2 or not ids.is_contiguous() or not ids.is_cuda:
        raise ValueError("ids must be a contiguous [tokens, top] matrix of int32 or int64 on a GPU")
    tokens, top = ids.shape
    size = _lib.ozb_expert_sort_rows(tokens, top, experts, align) if max(ids.numel(), experts, align) <= _MOST else -1
    if size < 0:
        raise ValueError(f"cannot sort {tokens} x {top} slots over {experts} experts in segments of {align}: sizes are positive, at most 1024 experts, align at most 256")
    need = _lib.ozb_expert_sort_scratch(tokens, top, experts)
    offsets, rows, slots = ids.new_empty(experts + 1, dtype=torch.int32), ids.new_empty(tokens, top, dtype=torch.int32), ids.new_empty(size, dtype=torch.int32)
    scratch = ids.new_empty(need, dtype=torch.uint8) if need else None
    _call(ids.get_device(), _lib.ozb_expert_sort, tokens, top, experts, ids.data_ptr(), ids.element_size(), align, size, offsets.data_ptr(), rows.data_ptr(),
          slots.data_ptr(), scratch.data_ptr() if need else None, need)
    return Routing(offsets, rows, slots, align)


def gather(x, routing, out=None):
    """The rows of x [T, h] in the order of their experts, [R, h]; zeros where a row has no slot."""
    ldx, index = _pitch(x, "x"), x.get_device()
    tokens, top = _routed(routing, index)
    if x.shape[0] != tokens:
        raise ValueError(f"x has {x.shape[0]} rows, the routing {tokens} tokens")
    if x.requires_grad:
        _cut("gather")
    kind, r, h = _type(x.dtype), routing.slots.shape[0], x.shape[1]
    y, ldy = _result(x, out, (r, h), x.dtype)
    _call(index, _lib.ozb_expert_gather, tokens, top, h, x.data_ptr(), kind, ldx, r, routing.rows.data_ptr(), routing.slots.data_ptr(), y.data_ptr(), ldy)
    return y


def combine(z, routing, weights=None, out=None):
    """y[t] = sum over j of weights[t, j] z[rows[t, j]] (weights None: 1), in FP32, rounded once to z's type. z has all of the routing's rows."""
    ldz, index = _pitch(z, "z"), z.get_device()
    tokens, top = _routed(routing, index)
    kind, (r, h), w = _type(z.dtype), z.shape, _weights(weights, routing.rows.shape, index)
    if r < routing.slots.shape[0]:
        raise ValueError(f"z has {r} rows, the routing {routing.slots.shape[0]} rows")
    if z.requires_grad or w is not None and weights.requires_grad:
        _cut("combine")
    y, ldy = _result(z, out, (tokens, h), z.dtype)
    _call(index, _lib.ozb_expert_combine, tokens, top, h, z.data_ptr(), kind, r, ldz, routing.rows.data_ptr(), w, y.data_ptr(), ldy)
    return y


def combine_grad(dy, z, routing, weights=None):
    """(dz, dweights) of combine(z, routing, weights) for a gradient dy [T, h] of z's type; dz is zero where a row has no slot."""
    lddy, ldz, index = _pitch(dy, "dy"), _pitch(z, "z"), z.get_device()
    tokens, top = _routed(routing, index)
    r, h = z.shape
    if dy.dtype is not z.dtype or dy.shape != (tokens, h) or r != routing.slots.shape[0] or dy.get_device() != index:
        raise ValueError(f"dy {tuple(dy.shape)} of {dy.dtype} and z {tuple(z.shape)} of {z.dtype} do not fit a routing of {tokens} tokens and {routing.slots.shape[0]} rows")
    kind, w = _type(z.dtype), _weights(weights, routing.rows.shape, index)
    if dy.requires_grad or z.requires_grad or w is not None and weights.requires_grad:
        _cut("combine_grad")
    dz, dweights = z.new_empty(r, h), z.new_empty(tokens, top, dtype=torch.float32)
    _call(index, _lib.ozb_expert_combine_grad, tokens, top, h, dy.data_ptr(), kind, lddy, z.data_ptr(), ldz, r, routing.rows.data_ptr(),
          routing.slots.data_ptr(), w, dz.data_ptr(), h, dweights.data_ptr())
    return dz, dweights


def matmul(x, w, ids, weights=None, keep=False):
    """y[t] = sum over j of weights[t, j] W[ids[t, j]] x[t]: tokens sorted by expert, rounded to the 4-bit format as they are gathered, one
    product for all experts, and the rows added up by token, in one call of the library. w: Mx4 stack [experts, n, ...] with blocks
    along the rows of x. keep: returns (y, z, routing) for matmul_grad, with segments padded to 64; z's rows behind the last segment are not written."""
    ldx, index = _pitch(x, "x"), x.get_device()
    kind, (tokens, k) = _type(x.dtype), x.shape
    if (ids.dtype is not torch.int32 and ids.dtype is not torch.int64) or ids.dim() != 2 or ids.shape[0] != tokens or not ids.is_contiguous() or ids.get_device() != index or ids.numel() > _MOST:
        raise ValueError(f"ids must be a contiguous [{tokens}, top] matrix of int32 or int64 on cuda:{index}")
    wc, ldw, ws, ldws = _codes(w, "w", 3, index)
    if w.length != k:
        raise ValueError(f"cannot multiply rows of {k} by vectors of {w.length}")
    (experts, n), top = w.codes.shape[:2], ids.shape[1]
    factors = _weights(weights, ids.shape, index)
    if x.requires_grad or factors is not None and weights.requires_grad:
        _cut("matmul")
    align = 64 if keep else 1
    need = _lib.ozb_expert_mx4_work(tokens, top, experts, n, k, kind, align)
    if not need:
        raise ValueError(f"cannot sort {tokens} x {top} slots over {experts} experts: sizes are positive, at most 1024 experts")
    y, work = x.new_empty(tokens, n), x.new_empty(need, dtype=torch.uint8)
    maps, z, r = (None, None, None, None), None, None
    if keep:
        size = _lib.ozb_expert_sort_rows(tokens, top, experts, align)
        r = Routing(ids.new_empty(experts + 1, dtype=torch.int32), ids.new_empty(tokens, top, dtype=torch.int32), ids.new_empty(size, dtype=torch.int32), align)
        z = x.new_empty(size, n)
        maps = r.offsets.data_ptr(), r.rows.data_ptr(), r.slots.data_ptr(), z.data_ptr()
    _call(index, _lib.ozb_expert_mx4, tokens, top, experts, n, k, x.data_ptr(), kind, ldx, ids.data_ptr(), ids.element_size(), factors, wc, ldw,
          w.codes.stride(0), ws, ldws, w.scales.stride(0), align, *maps, n, y.data_ptr(), n, work.data_ptr(), need)
    return (y, z, r) if keep else y


def matmul_grad(dy, x, z, wt, routing, weights=None):
    """The gradients of matmul(..., keep=True): (dx, dweights, dw) with dw [experts, n, k] of x's type, in one call of the library. wt: the
    weights with blocks along n, mx4.quantize(W, dim=-2), a stack [experts, k, ...]. Operands of the products are rounded to the 4-bit
    format, gradients pass through that rounding. dw of an expert whose segment is not padded to 64, which only a Routing of unknown
    padding can bring here, is NaN."""
    if routing.align % 64:
        raise ValueError(f"the segments are padded to {routing.align}: products along the tokens need multiples of 64 (matmul with keep=True)")
    lddy, ldx, ldz, index = _pitch(dy, "dy"), _pitch(x, "x"), _pitch(z, "z"), x.get_device()
    tokens, top = _routed(routing, index)
    kind, (r, n), k = _type(x.dtype), z.shape, x.shape[1]
    wc, ldw, ws, ldws = _codes(wt, "wt", 3, index)
    experts = wt.codes.shape[0]
    if not dy.dtype is z.dtype is x.dtype or dy.shape != (tokens, n) or x.shape[0] != tokens or r != routing.slots.shape[0] or dy.get_device() != index or z.get_device() != index:
        raise ValueError(f"dy {tuple(dy.shape)}, x {tuple(x.shape)} and z {tuple(z.shape)} do not fit a routing of {tokens} tokens and {routing.slots.shape[0]} rows, or differ in type")
    if _offsets(routing.offsets, index) != experts or wt.length != n or wt.codes.shape[1] != k:
        raise ValueError(f"wt must be a stack of {routing.offsets.shape[0] - 1} matrices of {k} vectors of {n}")
    factors = _weights(weights, routing.rows.shape, index)
    if dy.requires_grad or x.requires_grad or z.requires_grad or factors is not None and weights.requires_grad:
        _cut("matmul_grad")
    need = _lib.ozb_expert_mx4_grad_work(r, n, k, kind)
    dx, dweights = x.new_empty(tokens, k), x.new_empty(tokens, top, dtype=torch.float32)
    dw, work = x.new_empty(experts, n, k), x.new_empty(need, dtype=torch.uint8)
    _call(index, _lib.ozb_expert_mx4_grad, tokens, top, experts, n, k, r, dy.data_ptr(), kind, lddy, x.data_ptr(), ldx, z.data_ptr(), ldz, wc, ldw,
          wt.codes.stride(0), ws, ldws, wt.scales.stride(0), routing.offsets.data_ptr(), routing.rows.data_ptr(), routing.slots.data_ptr(), factors,
          dx.data_ptr(), k, dweights.data_ptr(), dw.data_ptr(), k, n * k, work.data_ptr(), need)
    return dx, dweights, dw
