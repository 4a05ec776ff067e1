"""A frozen LM head in 8-bit integers: half the weight to read, twice the matrix rate.

    z[t, v] = s_t * scale[v] * sum_i q[t, i] * values[v, i],      q = round(127 x / max |x|), s = max |x| / 127 of a hidden row x

* ``quantize_head`` -- the weight as int8 values with one fp32 scale a vocabulary row, laid out once;
* ``int8_logits`` -- the logits of a decoding step, for a sampler, ``torch_utils.top_logprobs_from_logits`` or ``beam_search.beam_select``;
* ``int8_logprobs_from_hidden`` -- log-probability and entropy of given tokens without a ``[T, V]`` tensor: scoring with a reference model.

The hidden states are brought to integers inside the call, a scale a token (ties to even; the quotients are rounded as if they were exact).  Sums of
products are exact; with weights and hidden states rounded to a step of max / 127, logits are those of the rounded operands to fp32 precision.  Neither
has a gradient.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Tuple

import torch

from . import _lib
from ._launch import call, device_guard, has_tangent, raw_stream, registered_op
from .ops import _require_device

__all__ = ["Int8Head", "quantize_head", "int8_logits", "int8_logprobs_from_hidden", "lmhead_int8_rows", "lmhead_int8_fwd", "lmhead_int8_logits"]

MAX_HIDDEN = 132096  # the largest sum of products, 127 * 128 * H, stays below 2^31
_K = 128             # rows of values are whole multiples of this long
_DTYPES = {torch.bfloat16: 0, torch.float32: 1}


class Int8Head(NamedTuple):
    """``weight[v, i] = scale[v] * values[v, i]``: ``values`` int8 ``[V, H rounded up to a multiple of 128]`` (what lies behind ``H`` does not enter),
    ``scale`` fp32 ``[V]``.  ``quantize_head`` makes one; the tensors of an 8-bit checkpoint are one, filled up where ``H`` is not such a multiple."""

    values: torch.Tensor
    scale: torch.Tensor


def _padded(hidden_size: int) -> int:
    return -(-hidden_size // _K) * _K


def _pitch(rows: torch.Tensor) -> int:
    return int(rows.stride(0) if rows.shape[0] > 1 else rows.shape[1])


def _check_rows(name: str, rows: torch.Tensor) -> None:
    if rows.dim() != 2:
        raise ValueError(f"expected {name} of two dimensions, got {tuple(rows.shape)}")
    if rows.dtype not in _DTYPES:
        raise TypeError(f"{name} must be torch.bfloat16 or torch.float32, got {rows.dtype}")
    if not 1 <= rows.shape[1] <= MAX_HIDDEN:
        raise ValueError(f"{name} rows must have 1 to {MAX_HIDDEN} elements, got {tuple(rows.shape)}")
    if rows.shape[1] > 1 and rows.stride(1) != 1 or _pitch(rows) < rows.shape[1]:
        raise ValueError(f"{name} must have unit stride in the last dimension and rows that do not overlap")


def _check_head(values: torch.Tensor, scale: torch.Tensor, hidden_size: int) -> int:
    """The vocabulary's size."""
    if values.dim() != 2 or scale.dim() != 1 or values.shape[0] != scale.shape[0] or values.shape[1] != _padded(hidden_size):
        raise ValueError(f"expected values [V, {_padded(hidden_size)}] and scale [V] for hidden states of {hidden_size}, got {tuple(values.shape)} and "
                         f"{tuple(scale.shape)}")
    if values.dtype != torch.int8 or scale.dtype != torch.float32:
        raise TypeError(f"values must be int8 and scale fp32, got {values.dtype} and {scale.dtype}")
    if values.stride(1) != 1 or _pitch(values) < values.shape[1] or not scale.is_contiguous():
        raise ValueError("values must have unit stride in the last dimension and rows that do not overlap, and scale must be contiguous")
    if values.shape[0] < 1:
        raise ValueError("a head needs at least one vocabulary row")
    return int(values.shape[0])


@registered_op("skyrl_amd::lmhead_int8_rows", mutates_args=())
def lmhead_int8_rows(rows: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(values int8 [n, H rounded up to a multiple of 128], scale fp32 [n])`` of ``rows [n, H]``."""
    _check_rows("the matrix", rows)
    dev = _require_device(rows)
    n, H = (int(x) for x in rows.shape)
    values, scale = torch.empty((n, _padded(H)), dtype=torch.int8, device=dev), torch.empty(n, dtype=torch.float32, device=dev)
    if n == 0:
        return values, scale
    with device_guard(dev):
        st = _lib.load().skyrl_lmhead_int8_rows(rows.data_ptr(), _DTYPES[rows.dtype], _pitch(rows), n, H, values.data_ptr(), values.shape[1], scale.data_ptr(),
                                                raw_stream(dev))
    _lib.check(st, "skyrl_lmhead_int8_rows")
    return values, scale


@lmhead_int8_rows.register_fake
def _(rows):
    return rows.new_empty((rows.shape[0], _padded(rows.shape[1])), dtype=torch.int8), rows.new_empty(rows.shape[0], dtype=torch.float32)


def _workspace(nbytes: int, dev: torch.device, what: str) -> torch.Tensor:
    if nbytes == 0:
        raise ValueError(f"no workspace for {what}: an extent is out of range")
    return torch.empty(nbytes, dtype=torch.uint8, device=dev)


@registered_op("skyrl_amd::lmhead_int8_logits", mutates_args=())
def lmhead_int8_logits(hidden: torch.Tensor, values: torch.Tensor, scale: torch.Tensor, fp32: bool) -> torch.Tensor:
    """Logits ``[T, V]``, bf16 or fp32."""
    _check_rows("hidden", hidden)
    T, H = (int(x) for x in hidden.shape)
    V = _check_head(values, scale, H)
    dev = _require_device(hidden, values, scale)
    out = torch.empty((T, V), dtype=torch.float32 if fp32 else torch.bfloat16, device=dev)
    if T == 0:
        return out
    lib = _lib.load()
    ws = _workspace(int(lib.skyrl_lmhead_int8_logits_workspace_bytes(T, H)), dev, f"T={T}, H={H}")
    with device_guard(dev):
        st = lib.skyrl_lmhead_int8_logits(hidden.data_ptr(), _DTYPES[hidden.dtype], _pitch(hidden), values.data_ptr(), _pitch(values), scale.data_ptr(), T, H, V,
                                          int(fp32), out.data_ptr(), V, ws.data_ptr(), ws.numel(), raw_stream(dev))
    _lib.check(st, "skyrl_lmhead_int8_logits")
    return out


@lmhead_int8_logits.register_fake
def _(hidden, values, scale, fp32):
    return hidden.new_empty((hidden.shape[0], values.shape[0]), dtype=torch.float32 if fp32 else torch.bfloat16)


@registered_op("skyrl_amd::lmhead_int8_fwd", mutates_args=())
def lmhead_int8_fwd(hidden: torch.Tensor, values: torch.Tensor, scale: torch.Tensor, labels: torch.Tensor, rcp_temperature: float, want_entropy: bool
                    ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(logprobs, entropy)``, fp32 ``[T]``; without ``want_entropy`` the entropy comes back empty (0 elements) and costs nothing."""
    _check_rows("hidden", hidden)
    T, H = (int(x) for x in hidden.shape)
    V = _check_head(values, scale, H)
    if labels.dtype != torch.int64 or labels.shape != (T,) or not labels.is_contiguous():
        raise ValueError(f"labels must be a contiguous int64 tensor of shape [{T}], got {labels.dtype} {tuple(labels.shape)}")
    dev = _require_device(hidden, values, scale, labels)
    logprobs, entropy = torch.empty(T, dtype=torch.float32, device=dev), torch.empty(T if want_entropy else 0, dtype=torch.float32, device=dev)
    if T == 0:
        return logprobs, entropy
    lib = _lib.load()
    ws = _workspace(int(lib.skyrl_lmhead_int8_fwd_workspace_bytes(T, H, V)), dev, f"T={T}, H={H}, V={V}")
    with device_guard(dev):
        st = lib.skyrl_lmhead_int8_fwd(hidden.data_ptr(), _DTYPES[hidden.dtype], _pitch(hidden), values.data_ptr(), _pitch(values), scale.data_ptr(),
                                       labels.data_ptr(), T, H, V, float(rcp_temperature), logprobs.data_ptr(), entropy.data_ptr() if want_entropy else None,
                                       ws.data_ptr(), ws.numel(), raw_stream(dev))
    _lib.check(st, "skyrl_lmhead_int8_fwd")
    return logprobs, entropy


@lmhead_int8_fwd.register_fake
def _(hidden, values, scale, labels, rcp_temperature, want_entropy):
    T = hidden.shape[0]
    return hidden.new_empty(T, dtype=torch.float32), hidden.new_empty(T if want_entropy else 0, dtype=torch.float32)


def quantize_head(weight: torch.Tensor) -> Int8Head:
    """``weight [V, H]`` (bf16 or fp32, rows of any pitch) as an ``Int8Head``.  A row with NaN or an infinity among its elements has a scale of NaN, and so
    logits of NaN."""
    with torch.no_grad():
        return Int8Head(*call(lmhead_int8_rows, weight.detach()))


def _rows(hidden: torch.Tensor) -> torch.Tensor:
    if hidden.dim() < 1 or hidden.shape[-1] == 0:
        raise ValueError(f"hidden must have a last dimension of one element or more, got {tuple(hidden.shape)}")
    rows = hidden.reshape(-1, hidden.shape[-1])
    fine = (rows.shape[1] <= 1 or rows.stride(1) == 1) and _pitch(rows) >= rows.shape[1]
    return rows if fine else rows.contiguous()


def _refuse_gradients(what: str, *operands: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in operands) or has_tangent(*operands):
        raise ValueError(f"{what} has no gradient: call it under torch.no_grad()")


def int8_logits(hidden: torch.Tensor, head: Int8Head, *, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Logits ``hidden.shape[:-1] + (V,)`` in ``dtype`` (bf16 or fp32) of ``hidden [..., H]`` (bf16 or fp32).  A hidden row with NaN or an infinity has
    logits of NaN.  Not differentiable: operands that ask for a gradient are refused outside ``torch.no_grad()``."""
    if dtype not in _DTYPES:
        raise TypeError(f"logits are torch.bfloat16 or torch.float32, got {dtype}")
    values, scale = head
    _refuse_gradients("int8_logits", hidden, scale)
    with torch.no_grad():
        out = call(lmhead_int8_logits, _rows(hidden), values, scale, dtype == torch.float32)
    return out.reshape(hidden.shape[:-1] + (values.shape[0],))


def int8_logprobs_from_hidden(hidden: torch.Tensor, head: Int8Head, labels: torch.Tensor, *, temperature: float = 1.0, compute_entropy: bool = True
                              ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(logprobs, entropy)``, fp32 ``hidden.shape[:-1]``, of ``labels`` (outside ``[0, V)``: log-probability 0) under ``softmax(z / temperature)``; no ``[T, V]``
    tensor is formed.  With ``compute_entropy=False`` the entropy is an empty tensor and its sums are not formed.  Not differentiable: operands that
    ask for a gradient are refused outside ``torch.no_grad()``."""
    temperature = float(temperature)
    if not 0.0 < temperature < math.inf or not 0.0 < 1.0 / temperature <= 3.4028234663852886e38:
        raise ValueError(f"temperature must be finite and positive, got {temperature}")
    if labels.shape != hidden.shape[:-1]:
        raise ValueError(f"labels {tuple(labels.shape)} do not match hidden {tuple(hidden.shape)}")
    if labels.dtype.is_floating_point or labels.dtype == torch.bool:
        raise TypeError(f"labels must be integers, got {labels.dtype}")
    values, scale = head
    _refuse_gradients("int8_logprobs_from_hidden", hidden, scale)
    with torch.no_grad():
        lp, ent = call(lmhead_int8_fwd, _rows(hidden), values, scale, labels.reshape(-1).to(torch.int64).contiguous(), 1.0 / temperature, bool(compute_entropy))
    return lp.reshape(labels.shape), ent.reshape(labels.shape) if compute_entropy else ent
