"""The LM head with low-rank adapters of many requests.

Every token of a batch has an adapter of its own, or none, on top of one frozen output weight:

    z_t = W h_t + scaling[a] * B[a] (A[a] h_t),      a = adapter_ids[t]; a value outside [0, N) means no adapter

with ``lora_a [N, R, H]`` and ``lora_b [N, V, R]`` in bf16 (the stacked ``lora_A`` / ``lora_B`` weights of ``N`` adapters; ``R`` a multiple of 8,
at most 256 -- an adapter of a lower rank is filled up with zeros, see ``stack_adapters``) and ``scaling [N]`` in fp32 (alpha / rank).  Tokens may
come in any order; sequences one behind the other are the cheapest.

* ``adapter_logits`` -- the logits of a decoding step, for a sampler or for ``torch_utils.top_logprobs_from_logits``;
* ``adapter_logprobs_from_hidden`` -- log-probability and entropy of given tokens without a ``[T, V]`` tensor, with gradients to the hidden
  states and to every adapter: training of many adapters in one batch.  No gradient reaches the weight.

The base head's tiles carry the adapters' part in the same accumulators; ``A h`` is kept in fp32 precision as two bf16 terms.  A token's results
do not depend on the values of adapters that it does not have.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from ._launch import call, device_guard, has_tangent, raw_stream, registered_op
from .ops import _ptr, _require_device

__all__ = ["MAX_RANK", "stack_adapters", "adapter_logits", "adapter_logprobs_from_hidden", "lmhead_adapter_logits", "lmhead_adapter_fwd",
           "lmhead_adapter_bwd"]

MAX_RANK = 256  # SKYRL_LMHEAD_MAX_ADAPTER_RANK
_MAX_PITCH = 1 << 22  # elements between rows that the kernels can walk
_DTYPES = {torch.bfloat16: 0, torch.float32: 1}


def _check(hidden, weight, lora_a, lora_b, scaling, adapter_ids) -> Tuple[int, int, int, int, int]:
    """``(T, H, V, N, R)`` of operands that the kernels can walk."""
    if hidden.dim() != 2 or weight.dim() != 2 or lora_a.dim() != 3 or lora_b.dim() != 3 or scaling.dim() != 1 or adapter_ids.dim() != 1:
        raise ValueError("expected hidden [T,H], weight [V,H], lora_a [N,R,H], lora_b [N,V,R], scaling [N], adapter_ids [T]; got "
                         + ", ".join(str(tuple(t.shape)) for t in (hidden, weight, lora_a, lora_b, scaling, adapter_ids)))
    T, H = (int(x) for x in hidden.shape)
    V, N, R = int(weight.shape[0]), int(lora_a.shape[0]), int(lora_a.shape[1])
    if weight.shape[1] != H or tuple(lora_a.shape) != (N, R, H) or tuple(lora_b.shape) != (N, V, R) or scaling.shape[0] != N or adapter_ids.shape[0] != T:
        raise ValueError("shape mismatch: hidden {}, weight {}, lora_a {}, lora_b {}, scaling {}, adapter_ids {}".format(
            *(tuple(t.shape) for t in (hidden, weight, lora_a, lora_b, scaling, adapter_ids))))
    for name, t in (("hidden", hidden), ("weight", weight), ("lora_a", lora_a), ("lora_b", lora_b)):
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be torch.bfloat16, got {t.dtype}")
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must have unit stride in the last dimension")
    if scaling.dtype != torch.float32 or adapter_ids.dtype != torch.int64:
        raise TypeError(f"scaling must be fp32 and adapter_ids int64, got {scaling.dtype} and {adapter_ids.dtype}")
    if not scaling.is_contiguous() or not adapter_ids.is_contiguous():
        raise ValueError("scaling and adapter_ids must be contiguous")
    if N < 1 or not 8 <= R <= MAX_RANK or R % 8 != 0:
        raise ValueError(f"need at least one adapter of a rank that is a multiple of 8 and at most {MAX_RANK}, got {N} of rank {R}")
    return T, H, V, N, R


def _adapter_args(lora_a, lora_b, scaling, adapter_ids, N: int, R: int):
    V, H = lora_b.shape[1], lora_a.shape[2]  # the stride of a dimension of one may be anything
    return (lora_a.data_ptr(), lora_a.stride(0) if N > 1 else R * H, lora_a.stride(1), lora_b.data_ptr(), lora_b.stride(0) if N > 1 else V * R,
            _pitch(lora_b[0]), scaling.data_ptr(), adapter_ids.data_ptr(), N, R)


def _pitch(rows: torch.Tensor) -> int:
    return int(rows.stride(0) if rows.shape[0] > 1 else rows.shape[1])


def _workspace(lib, nbytes: int, dev: torch.device, what: str) -> torch.Tensor:
    if nbytes == 0:
        raise ValueError(f"no workspace for {what}: an extent is out of range")
    return torch.empty(nbytes, dtype=torch.uint8, device=dev)


@registered_op("skyrl_amd::lmhead_adapter_logits", mutates_args=())
def lmhead_adapter_logits(hidden: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, scaling: torch.Tensor,
                          adapter_ids: torch.Tensor, fp32: bool) -> torch.Tensor:
    """Logits ``[T, V]``, bf16 or fp32."""
    T, H, V, N, R = _check(hidden, weight, lora_a, lora_b, scaling, adapter_ids)
    dev = _require_device(hidden, weight, lora_a, lora_b, scaling, adapter_ids)
    out = torch.empty((T, V), dtype=torch.float32 if fp32 else torch.bfloat16, device=dev)
    if T == 0:
        return out
    lib = _lib.load()
    ws = _workspace(lib, int(lib.skyrl_lmhead_adapter_logits_workspace_bytes(T, H, N, R)), dev, f"T={T}, H={H}, N={N}, rank={R}")
    with device_guard(dev):
        st = lib.skyrl_lmhead_adapter_logits(hidden.data_ptr(), _pitch(hidden), weight.data_ptr(), _pitch(weight),
                                             *_adapter_args(lora_a, lora_b, scaling, adapter_ids, N, R), T, H, V, int(fp32), out.data_ptr(), V,
                                             ws.data_ptr(), ws.numel(), raw_stream(dev))
    _lib.check(st, "skyrl_lmhead_adapter_logits")
    return out


@lmhead_adapter_logits.register_fake
def _(hidden, weight, lora_a, lora_b, scaling, adapter_ids, fp32):
    return hidden.new_empty((hidden.shape[0], weight.shape[0]), dtype=torch.float32 if fp32 else torch.bfloat16)


@registered_op("skyrl_amd::lmhead_adapter_fwd", mutates_args=())
def lmhead_adapter_fwd(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                       scaling: torch.Tensor, adapter_ids: torch.Tensor, rcp_temperature: float
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(logprobs, entropy, row_lse, row_pz)``, each fp32 ``[T]``."""
    T, H, V, N, R = _check(hidden, weight, lora_a, lora_b, scaling, adapter_ids)
    if labels.dtype != torch.int64 or labels.shape != (T,) or not labels.is_contiguous():
        raise ValueError(f"labels must be a contiguous int64 tensor of shape [{T}], got {labels.dtype} {tuple(labels.shape)}")
    dev = _require_device(hidden, weight, labels, lora_a, lora_b, scaling, adapter_ids)
    lp, ent, lse, pz = (torch.empty(T, dtype=torch.float32, device=dev) for _ in range(4))
    if T == 0:
        return lp, ent, lse, pz
    lib = _lib.load()
    ws = _workspace(lib, int(lib.skyrl_lmhead_adapter_fwd_workspace_bytes(T, H, V, N, R)), dev, f"T={T}, H={H}, V={V}, N={N}, rank={R}")
    with device_guard(dev):
        st = lib.skyrl_lmhead_adapter_fwd(hidden.data_ptr(), _pitch(hidden), weight.data_ptr(), _pitch(weight), labels.data_ptr(),
                                          *_adapter_args(lora_a, lora_b, scaling, adapter_ids, N, R), T, H, V, float(rcp_temperature), lp.data_ptr(),
                                          ent.data_ptr(), lse.data_ptr(), pz.data_ptr(), ws.data_ptr(), ws.numel(), raw_stream(dev))
    _lib.check(st, "skyrl_lmhead_adapter_fwd")
    return lp, ent, lse, pz


@lmhead_adapter_fwd.register_fake
def _(hidden, weight, labels, lora_a, lora_b, scaling, adapter_ids, rcp_temperature):
    return tuple(hidden.new_empty(hidden.shape[0], dtype=torch.float32) for _ in range(4))


@registered_op("skyrl_amd::lmhead_adapter_bwd", mutates_args=())
def lmhead_adapter_bwd(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                       scaling: torch.Tensor, adapter_ids: torch.Tensor, row_lse: torch.Tensor, row_pz: Optional[torch.Tensor],
                       dlogprobs: torch.Tensor, dentropy: Optional[torch.Tensor], rcp_temperature: float
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(d_hidden [T, H], d_lora_a [N, R, H], d_lora_b [N, V, R])``, bf16, on the tokens that have an upstream gradient."""
    T, H, V, N, R = _check(hidden, weight, lora_a, lora_b, scaling, adapter_ids)
    if labels.dtype != torch.int64 or labels.shape != (T,) or not labels.is_contiguous():
        raise ValueError(f"labels must be a contiguous int64 tensor of shape [{T}], got {labels.dtype} {tuple(labels.shape)}")
    if dentropy is not None and row_pz is None:
        raise ValueError("a gradient on the entropy needs row_pz")
    for name, t in (("row_lse", row_lse), ("row_pz", row_pz), ("dlogprobs", dlogprobs), ("dentropy", dentropy)):
        if t is not None and (t.dtype != torch.float32 or t.shape != (T,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous fp32 tensor of shape [{T}], got {t.dtype} {tuple(t.shape)}")
    dev = _require_device(*[t for t in (hidden, weight, labels, lora_a, lora_b, scaling, adapter_ids, row_lse, row_pz, dlogprobs, dentropy)
                            if t is not None])
    b16 = dict(dtype=torch.bfloat16, device=dev)
    if T == 0:  # an empty micro-batch contributes zero gradients
        return torch.empty((T, H), **b16), torch.zeros((N, R, H), **b16), torch.zeros((N, V, R), **b16)
    dh, da, db = torch.empty((T, H), **b16), torch.empty((N, R, H), **b16), torch.empty((N, V, R), **b16)
    lib = _lib.load()
    ws = _workspace(lib, int(lib.skyrl_lmhead_adapter_bwd_workspace_bytes(T, H, V, N, R)), dev, f"T={T}, H={H}, V={V}, N={N}, rank={R}")
    with device_guard(dev):
        st = lib.skyrl_lmhead_adapter_bwd(hidden.data_ptr(), _pitch(hidden), weight.data_ptr(), _pitch(weight), labels.data_ptr(),
                                          *_adapter_args(lora_a, lora_b, scaling, adapter_ids, N, R), row_lse.data_ptr(), _ptr(row_pz),
                                          dlogprobs.data_ptr(), _ptr(dentropy), T, H, V, float(rcp_temperature), dh.data_ptr(), da.data_ptr(),
                                          db.data_ptr(), ws.data_ptr(), ws.numel(), raw_stream(dev))
    _lib.check(st, "skyrl_lmhead_adapter_bwd")
    return dh, da, db


@lmhead_adapter_bwd.register_fake
def _(hidden, weight, labels, lora_a, lora_b, scaling, adapter_ids, row_lse, row_pz, dlogprobs, dentropy, rcp_temperature):
    return tuple(t.new_empty(t.shape, dtype=torch.bfloat16) for t in (hidden, lora_a, lora_b))


class _AdapterLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels, lora_a, lora_b, scaling, adapter_ids, rcp_temperature):
        lp, ent, lse, pz = call(lmhead_adapter_fwd, hidden, weight, labels, lora_a, lora_b, scaling, adapter_ids, rcp_temperature)
        ctx.save_for_backward(hidden, weight, labels, lora_a, lora_b, scaling, adapter_ids, lse, pz)
        ctx.rcp_temperature = rcp_temperature
        ctx.set_materialize_grads(False)
        return lp, ent

    @staticmethod
    def backward(ctx, dlp, dent):
        if dlp is None and dent is None:
            return (None,) * 8
        *operands, lse, pz = ctx.saved_tensors
        f = lambda t: None if t is None else t.to(torch.float32).contiguous()  # noqa: E731
        g = torch.zeros_like(lse) if dlp is None else f(dlp)
        dh, da, db = call(lmhead_adapter_bwd, *operands, lse, None if dent is None else pz, g, f(dent), ctx.rcp_temperature)
        need = ctx.needs_input_grad
        return dh if need[0] else None, None, None, da if need[3] else None, db if need[4] else None, None, None, None


def _rows(hidden: torch.Tensor, adapter_ids: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    if adapter_ids.shape != hidden.shape[:-1]:
        raise ValueError(f"adapter_ids {tuple(adapter_ids.shape)} do not match hidden {tuple(hidden.shape)}")
    if adapter_ids.dtype.is_floating_point:
        raise TypeError(f"adapter_ids must be integers, got {adapter_ids.dtype}")
    rows = hidden.reshape(-1, hidden.shape[-1])
    if not rows.shape[1] <= _pitch(rows) <= _MAX_PITCH or _pitch(rows) % 8 != 0:
        rows = rows.contiguous()  # the last position of each long sequence, one row repeated, rows that do not begin on 16 bytes
    return rows, adapter_ids.reshape(-1).to(torch.int64).contiguous()


def adapter_logits(hidden: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, scaling: torch.Tensor,
                   adapter_ids: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Logits ``hidden.shape[:-1] + (V,)`` in ``dtype`` (bf16 or fp32) of ``hidden [..., H]`` with the adapters of ``adapter_ids [...]``.
    Not differentiable: operands that ask for a gradient are refused outside ``torch.no_grad()``, and those with a tangent; for training see
    ``adapter_logprobs_from_hidden``."""
    if dtype not in _DTYPES:
        raise TypeError(f"logits are torch.bfloat16 or torch.float32, got {dtype}")
    operands = (hidden, weight, lora_a, lora_b, scaling)
    if torch.is_grad_enabled() and any(t.requires_grad for t in operands) or has_tangent(*operands):
        raise ValueError("adapter_logits has no gradient: call it under torch.no_grad(), or adapter_logprobs_from_hidden for training")
    rows, ids = _rows(hidden, adapter_ids)
    with torch.no_grad():
        out = call(lmhead_adapter_logits, rows, weight, lora_a, lora_b, scaling, ids, dtype == torch.float32)
    return out.reshape(hidden.shape[:-1] + (weight.shape[0],))


def adapter_logprobs_from_hidden(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                                 scaling: torch.Tensor, adapter_ids: torch.Tensor, *, temperature: float = 1.0
                                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(logprobs, entropy)``, fp32 ``hidden.shape[:-1]``, of ``labels`` (outside ``[0, V)``: log-probability 0, without a gradient) under
    ``softmax(z / temperature)``.  Both carry gradients to ``hidden``, ``lora_a`` and ``lora_b`` (bf16); ``weight`` and ``scaling`` take none, and either that
    asks for one is refused."""
    temperature = float(temperature)
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"temperature must be finite and positive, got {temperature}")
    if torch.is_grad_enabled() and (weight.requires_grad or scaling.requires_grad):
        raise ValueError("the head with adapters is frozen: weight and scaling take no gradient")
    if labels.shape != hidden.shape[:-1]:
        raise ValueError(f"labels {tuple(labels.shape)} do not match hidden {tuple(hidden.shape)}")
    rows, ids = _rows(hidden, adapter_ids)
    lp, ent = _AdapterLogprobs.apply(rows, weight, labels.reshape(-1).to(torch.int64).contiguous(), lora_a, lora_b, scaling, ids, 1.0 / temperature)
    return lp.reshape(hidden.shape[:-1]), ent.reshape(hidden.shape[:-1])


def stack_adapters(pairs: Sequence[Tuple[torch.Tensor, torch.Tensor]], scaling: Sequence[float]
                   ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(lora_a, lora_b, scaling)`` as the operators take them from ``(lora_A [r, H], lora_B [V, r])`` pairs of any ranks: bf16, filled up with
    zeros to the largest rank, rounded up to a multiple of 8.  Differentiable with respect to the pairs."""
    if not pairs or len(pairs) != len(scaling):
        raise ValueError(f"need one scaling per adapter and at least one adapter, got {len(pairs)} and {len(scaling)}")
    rank = -(-max(int(a.shape[0]) for a, _ in pairs) // 8) * 8
    for a, b in pairs:
        if a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1] or a.shape[1] != pairs[0][0].shape[1] or b.shape[0] != pairs[0][1].shape[0]:
            raise ValueError("expected pairs of lora_A [r, H] and lora_B [V, r] with one H and V, got " + ", ".join(
                f"{tuple(x.shape)} and {tuple(y.shape)}" for x, y in pairs))
    pad = torch.nn.functional.pad
    lora_a = torch.stack([pad(a.to(torch.bfloat16), (0, 0, 0, rank - a.shape[0])) for a, _ in pairs])
    lora_b = torch.stack([pad(b.to(torch.bfloat16), (0, rank - b.shape[1])) for _, b in pairs])
    return lora_a, lora_b, torch.tensor(list(scaling), dtype=torch.float32, device=lora_a.device)
