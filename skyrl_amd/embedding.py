"""The embedding that a model begins with, and whose table is often the weight of its LM head.

    out[t] = scale * weight[ids[t]]                         zeros where ids[t] lies outside [0, V)
    d_weight[v] = scale * sum of d_out[t] over the tokens with ids[t] = v       zeros where v is the padding id

* ``embedding_lookup`` -- the rows, in the table's dtype (bf16 or fp32), with a gradient to the table;
* ``embedding_backward_accumulate`` -- the gradient added into an fp32 ``[V, H]`` buffer, next to ``ops.lmhead_bwd_accumulate``: a tied table's
  gradient from both of its uses, of which this one touches only the rows that the tokens name.

An id outside the table gives a row of zeros and takes no gradient, as a label outside a vocabulary shard has no log-probability here.  Sums are
formed in fp32 in an order that the ids fix, and rounded once: the same bits on each call.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.graph import increment_version

from . import _lib
from ._launch import call, device_guard, direct, has_tangent, raw_stream, registered_op
from .ops import _require_device

__all__ = ["embedding_lookup", "embedding_backward_accumulate", "lmhead_embedding_fwd", "lmhead_embedding_bwd"]

_DTYPES = {torch.bfloat16: 0, torch.float32: 1}
_NO_PADDING = -1


def _check_table(weight: torch.Tensor) -> None:
    if weight.dim() != 2 or weight.dtype not in _DTYPES:
        raise TypeError(f"the table must be a bf16 or fp32 matrix [V, H], got {weight.dtype} {tuple(weight.shape)}")
    (V, H), (row, column) = weight.shape, weight.stride()
    if column != 1 and H > 1 or row < H and V > 1:
        raise ValueError("the table must have unit stride in the last dimension and rows that do not overlap")


def _check_ids(ids: torch.Tensor) -> None:
    if ids.dtype != torch.int64 or ids.dim() != 1 or not ids.is_contiguous():
        raise ValueError(f"ids must be a contiguous int64 tensor of one dimension, got {ids.dtype} {tuple(ids.shape)}")


@registered_op("skyrl_amd::lmhead_embedding_fwd", mutates_args=())
def lmhead_embedding_fwd(weight: torch.Tensor, ids: torch.Tensor, scale: float) -> torch.Tensor:
    """``[T, H]`` in the table's dtype."""
    _check_table(weight)
    _check_ids(ids)
    dev = _require_device(weight, ids)
    (V, H), T = weight.shape, ids.shape[0]
    out = torch.empty((T, H), dtype=weight.dtype, device=dev)
    if T == 0 or H == 0:
        return out
    if V == 0:  # every id lies outside
        return out.zero_()
    with device_guard(dev):
        st = _lib.load().skyrl_lmhead_embedding_fwd(weight.data_ptr(), _DTYPES[weight.dtype], weight.stride(0) if V > 1 else H, ids.data_ptr(), T, H, V, scale,
                                                    out.data_ptr(), raw_stream(dev))
    _lib.check(st, "skyrl_lmhead_embedding_fwd")
    return out


@lmhead_embedding_fwd.register_fake
def _(weight, ids, scale):
    return weight.new_empty((ids.shape[0], weight.shape[1]))


def _backward_into(d_out: torch.Tensor, ids: torch.Tensor, scale: float, padding_idx: int, d_weight: torch.Tensor, accumulate: int) -> None:
    (T, H), V, dev = d_out.shape, d_weight.shape[0], d_out.device
    lib = _lib.load()
    nbytes = lib.skyrl_lmhead_embedding_bwd_workspace_bytes(T, H, V)
    if nbytes == 0:
        raise ValueError(f"no workspace for T={T}, H={H}, V={V}: an extent is out of range")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with device_guard(dev):
        st = lib.skyrl_lmhead_embedding_bwd(d_out.data_ptr(), _DTYPES[d_out.dtype], d_out.stride(0) if T > 1 else H, ids.data_ptr(), padding_idx, T, H, V, scale,
                                            accumulate, d_weight.data_ptr(), ws.data_ptr(), nbytes, raw_stream(dev))
    _lib.check(st, "skyrl_lmhead_embedding_bwd")


def _check_gradient(d_out: torch.Tensor, ids: torch.Tensor) -> None:
    if d_out.dim() != 2 or d_out.dtype not in _DTYPES:
        raise TypeError(f"the gradient of the rows must be a bf16 or fp32 matrix [T, H], got {d_out.dtype} {tuple(d_out.shape)}")
    _check_ids(ids)
    if ids.shape[0] != d_out.shape[0]:
        raise ValueError(f"ids {tuple(ids.shape)} do not match the gradient {tuple(d_out.shape)}")
    if d_out.stride(1) != 1 and d_out.shape[1] > 1 or d_out.shape[0] > 1 and 0 < d_out.stride(0) < d_out.shape[1]:
        raise ValueError("the gradient of the rows must have unit stride in the last dimension and rows that do not overlap")


@registered_op("skyrl_amd::lmhead_embedding_bwd", mutates_args=())
def lmhead_embedding_bwd(d_out: torch.Tensor, ids: torch.Tensor, vocab: int, scale: float, padding_idx: int) -> torch.Tensor:
    """``d_weight [vocab, H]`` in the dtype of ``d_out [T, H]``, of whatever strides; ``padding_idx``: -1 where there is none."""
    if d_out.dim() == 2:
        d_out = _walkable(d_out)
    _check_gradient(d_out, ids)
    if vocab < 0:
        raise ValueError(f"a table of {vocab} rows")
    dev = _require_device(d_out, ids)
    T, H = d_out.shape
    if T == 0 or H == 0 or vocab == 0:
        return torch.zeros((vocab, H), dtype=d_out.dtype, device=dev)
    d_weight = torch.empty((vocab, H), dtype=d_out.dtype, device=dev)
    _backward_into(d_out, ids, scale, padding_idx, d_weight, 0)
    return d_weight


@lmhead_embedding_bwd.register_fake
def _(d_out, ids, vocab, scale, padding_idx):
    return d_out.new_empty((vocab, d_out.shape[1]))


class _Lookup(torch.autograd.Function):
    """What csrc/lookup_node.cpp is to a plain eager call: the same over the ops, where anything follows the call."""

    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.rest = (weight.shape[0], scale, padding_idx)
        return lmhead_embedding_fwd(weight, ids, scale)

    @staticmethod
    def backward(ctx, d_out):
        (ids,) = ctx.saved_tensors
        return lmhead_embedding_bwd(d_out, ids, *ctx.rest), None, None, None


def _walkable(rows: torch.Tensor) -> torch.Tensor:
    T, H = rows.shape
    row, column = rows.stride()
    return rows if (column == 1 or H <= 1) and (row >= H or row == 0 or T <= 1) else rows.contiguous()


def _flat_ids(ids: torch.Tensor) -> torch.Tensor:
    if ids.dtype != torch.int64:
        if ids.dtype != torch.int32:
            raise TypeError(f"ids must be int64 or int32, got {ids.dtype}")
        ids = ids.to(torch.int64)
    return ids if ids.dim() == 1 and ids.is_contiguous() else ids.reshape(-1).contiguous()


def _scale_of(scale: float) -> float:
    scale = float(scale)
    if not math.isfinite(scale) or abs(scale) > 3.4028234663852886e38:
        raise ValueError(f"scale must be finite in fp32, got {scale}")
    return scale


def _padding_of(padding_idx: Optional[int], vocab: int) -> int:
    if padding_idx is None:
        return _NO_PADDING
    padding_idx = int(padding_idx)
    if not -vocab <= padding_idx < vocab:
        raise ValueError(f"padding_idx {padding_idx} lies outside a table of {vocab} rows")
    return padding_idx % vocab


def embedding_lookup(weight: torch.Tensor, ids: torch.Tensor, *, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[ids]``, shape ``ids.shape + (H,)``, in the dtype of ``weight [V, H]`` (bf16 or fp32; the product is formed in fp32 and
    rounded once).  ``ids`` are int64 or int32; one outside ``[0, V)`` gives zeros and takes no gradient.  ``padding_idx``: the row that takes none
    either, as in ``torch.nn.functional.embedding``.  The gradient is dense, ``[V, H]`` in the table's dtype.  At most 2^24 tokens."""
    _check_table(weight)
    flat, scale, padding_idx = _flat_ids(ids), _scale_of(scale), _padding_of(padding_idx, weight.shape[0])
    tangent = has_tangent(weight)
    if torch.is_grad_enabled() and weight.requires_grad or tangent:
        if direct(weight, flat, recorded=True) and not tangent:
            _require_device(weight, flat)
            rows = _lib.load_node().lookup(weight, flat, scale, padding_idx)
        else:
            rows = _Lookup.apply(weight, flat, scale, padding_idx)
    else:
        rows = call(lmhead_embedding_fwd, weight, flat, scale)
    return rows if flat is ids else rows.reshape(ids.shape + (weight.shape[1],))


def _meets(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the ranges of addresses of two tensors meet."""
    def reach(t):
        begin = t.data_ptr()
        return begin, begin + (t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) if t.numel() else 0)
    (a0, a1), (b0, b1) = reach(a), reach(b)
    return a0 < b1 and b0 < a1


def embedding_backward_accumulate(d_out: torch.Tensor, ids: torch.Tensor, d_weight_accum: torch.Tensor, *, scale: float = 1.0,
                                  padding_idx: Optional[int] = None) -> torch.Tensor:
    """Adds the gradient of ``embedding_lookup`` for the upstream gradient ``d_out`` (``ids.shape + (H,)``, bf16 or fp32) into ``d_weight_accum``, a
    contiguous fp32 ``[V, H]`` buffer in memory of its own, and returns it.  Rows that no token names are neither read nor written.  It works on addresses: a compiled program is
    left for the call and goes on behind it."""
    if d_weight_accum.dim() != 2 or d_weight_accum.dtype != torch.float32 or not d_weight_accum.is_contiguous():
        raise ValueError(f"d_weight_accum must be a contiguous fp32 matrix [V, H], got {d_weight_accum.dtype} {tuple(d_weight_accum.shape)}")
    if tuple(d_out.shape) != tuple(ids.shape) + (d_weight_accum.shape[1],):
        raise ValueError(f"d_out {tuple(d_out.shape)} does not match ids {tuple(ids.shape)} and d_weight_accum {tuple(d_weight_accum.shape)}")
    flat, scale, padding_idx = _flat_ids(ids), _scale_of(scale), _padding_of(padding_idx, int(d_weight_accum.shape[0]))
    if torch.is_grad_enabled() and d_weight_accum.requires_grad:
        raise ValueError("d_weight_accum is written in place and takes no gradient itself")
    rows = _walkable(d_out.detach().resolve_neg().reshape(flat.shape[0], d_weight_accum.shape[1]))
    _check_gradient(rows, flat)
    if _meets(rows, d_weight_accum) or _meets(flat, d_weight_accum):
        raise ValueError("d_weight_accum shares memory with d_out or the ids: it would be written while they are read")
    _require_device(rows, flat, d_weight_accum)
    if rows.numel() and d_weight_accum.numel():
        _backward_into(rows, flat, scale, padding_idx, d_weight_accum, 1)
        increment_version(d_weight_accum)
    return d_weight_accum
