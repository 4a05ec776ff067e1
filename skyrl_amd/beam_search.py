"""One step of beam search: the best continuations of each prompt's beams, and the beams' states brought to their order.

    total[n, b, v] = scores[n, b] + log_softmax(logits[n, b] / temperature)[v]

* ``beam_select`` -- the ``k`` largest totals of each prompt over beams and vocabulary, with the beam (``parents``) and the token of each;
* ``beam_reorder`` -- key / value caches and whatever else a beam carries follow their parents, into other buffers or in place, all tensors of a
  layout in one launch.

Among equal totals the lower beam and then the lower token comes first.  Totals are formed in 64 bits from exponentials that are right to a unit of their
last place in 32, so that candidates of different beams come in the order of their exact totals but where those differ by less than 2.4e-7 (or, under scores of
1e6 and more, than 2^-45 of them); candidates of one beam come in the order of their logits whatever its score is.  Neither waits for the GPU, and both may be
captured in a HIP graph.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import List, NamedTuple, Optional, Sequence, Tuple

import torch
from torch.autograd.graph import increment_version

from . import _lib
from ._launch import call, device_guard, has_tangent, raw_stream, registered_op
from .ops import _require_device

__all__ = ["MAX_CANDIDATES", "MAX_BEAMS", "BeamSelection", "beam_select", "beam_reorder", "logits_beam_select"]

MAX_CANDIDATES = 128  # SKYRL_LOGITS_TOP_MAX
MAX_BEAMS = 128       # SKYRL_LOGITS_BEAMS_MAX
_MAX_STATES = 200     # SKYRL_LOGITS_STATES_MAX
_DTYPES = {torch.bfloat16: 0, torch.float32: 1}


class BeamSelection(NamedTuple):
    scores: torch.Tensor   # [N, k] fp32, best first
    parents: torch.Tensor  # [N, k] int64, the beam that a candidate continues
    tokens: torch.Tensor   # [N, k] int64


def _check_select(logits: torch.Tensor, scores: torch.Tensor, k: int) -> Tuple[int, int, int]:
    if logits.dim() != 3:
        raise ValueError(f"expected logits [N, B, V], got {tuple(logits.shape)}")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be torch.bfloat16 or torch.float32, got {logits.dtype}")
    N, B, V = logits.shape
    if scores.shape != (N, B):
        raise ValueError(f"scores {tuple(scores.shape)} do not match logits {tuple(logits.shape)}")
    if scores.dtype != torch.float32:
        raise TypeError(f"scores must be torch.float32, got {scores.dtype}")
    if not 1 <= B <= MAX_BEAMS or not 1 <= k <= min(B * V, MAX_CANDIDATES):
        raise ValueError(f"need 1 to {MAX_BEAMS} beams and k from 1 to the candidates of a prompt and at most {MAX_CANDIDATES}, got {B} beams, V={V} and k={k}")
    return N, B, V


@registered_op("skyrl_amd::logits_beam_select", mutates_args=())
def logits_beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int, rcp_temperature: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(scores, parents, tokens)``, each ``[N, k]``, of ``logits [N, B, V]`` with unit stride along ``V`` and contiguous ``scores [N, B]``."""
    N, B, V = _check_select(logits, scores, k)
    if V > 1 and logits.stride(2) != 1 or not scores.is_contiguous():
        raise ValueError("logits must have unit stride in the last dimension and scores must be contiguous")
    dev = _require_device(logits, scores)
    best = torch.empty((N, k), dtype=torch.float32, device=dev)
    parents, tokens = (torch.empty((N, k), dtype=torch.int64, device=dev) for _ in range(2))
    if N == 0:
        return best, parents, tokens
    lib = _lib.load()
    nbytes = int(lib.skyrl_logits_beam_select_workspace_bytes(N, B, V, k))
    if nbytes == 0:
        raise ValueError(f"no workspace for N={N}, B={B}, V={V}, k={k}: an extent is out of range")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with device_guard(dev):
        st = lib.skyrl_logits_beam_select(logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0), logits.stride(1), scores.data_ptr(), N, B, V, k,
                                          float(rcp_temperature), best.data_ptr(), parents.data_ptr(), tokens.data_ptr(), ws.data_ptr(), nbytes, raw_stream(dev))
    _lib.check(st, "skyrl_logits_beam_select")
    return best, parents, tokens


@logits_beam_select.register_fake
def _(logits, scores, k, rcp_temperature):
    N = logits.shape[0]
    return scores.new_empty((N, k)), scores.new_empty((N, k), dtype=torch.int64), scores.new_empty((N, k), dtype=torch.int64)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int, *, temperature: float = 1.0) -> BeamSelection:
    """The ``k`` best candidates of each prompt, best first, of ``logits [N, B, V]`` (bf16 or fp32; rows of any pitch, shared by beams where the tensor is
    expanded) and the beams' ``scores [N, B]`` (fp32, the sums of their log-probabilities so far).

    ``k`` is at most 128 and may exceed the number of beams, as it has to where ended beams are set aside.  A beam of score -inf has ended; it, and one
    with no logit above -inf, offers tokens 0, 1, ... with a total of -inf.  One with a NaN or +inf among its logits, or whose score is NaN or +inf,
    offers the same with NaN, behind those.  Not differentiable: operands that ask for a gradient are refused outside ``torch.no_grad()``."""
    k, temperature = int(k), float(temperature)
    if not 0.0 < temperature < math.inf:
        raise ValueError(f"temperature must be finite and positive, got {temperature}")
    if torch.is_grad_enabled() and (logits.requires_grad or scores.requires_grad) or has_tangent(logits, scores):
        raise ValueError("beam_select has no gradient: call it under torch.no_grad()")
    rows = logits if logits.dim() != 3 or logits.shape[2] <= 1 or logits.stride(2) == 1 else logits.contiguous()
    scores = scores if scores.is_contiguous() else scores.contiguous()
    with torch.no_grad():
        return BeamSelection(*call(logits_beam_select, rows, scores, k, 1.0 / temperature))


_NOT_ITS_VALUE = "a state whose memory is not its value (a negative or conjugate view): resolve it first"


def _segments(shape: Tuple[int, ...], strides: Tuple[int, ...], to_strides: Tuple[int, ...], size: int) -> List[Tuple[int, int, int, int, int, int]]:
    """``(place, place in the result, segments, bytes, from_segment, to_segment)``, in bytes, of a row of that shape: what it is in both, one run of
    equally spaced contiguous pieces.  Rows with more dimensions that do not join are taken apart along the first of them."""
    dims: List[List[int]] = []  # [extent, stride, stride in the result], outer first, neighbours joined
    for n, x, y in zip(shape, strides, to_strides):
        if n == 1:
            continue
        if dims and dims[-1][1] == n * x and dims[-1][2] == n * y:
            dims[-1] = [dims[-1][0] * n, x, y]
        else:
            dims.append([n, x, y])
    inner = dims.pop()[0] if dims and dims[-1][1] == dims[-1][2] == 1 else 1
    if len(dims) > 1:
        axis = next(i for i, n in enumerate(shape) if n != 1)
        rest = _segments(shape[axis + 1:], strides[axis + 1:], to_strides[axis + 1:], size)
        return [(i * strides[axis] * size + at, i * to_strides[axis] * size + to_at, *more) for i in range(shape[axis]) for at, to_at, *more in rest]
    n, x, y = dims[0] if dims else (1, 0, 0)
    return [(0, 0, n, inner * size, x * size, y * size)]


def _folded(shape: Tuple[int, ...], strides: Tuple[int, ...]) -> bool:
    end = 0  # of the dimensions so far, the closest elements first
    for step, n in sorted((s, n) for n, s in zip(shape, strides) if n > 1):
        if step <= end:
            return True
        end += (n - 1) * step
    return False


def _in_memory_order(shape: Tuple[int, ...], strides: Tuple[int, ...], to_strides: Tuple[int, ...]) -> Tuple[Tuple[int, ...], ...]:
    """The dimensions of a row as the result has them in memory, outer first, which is where neighbours join; of several that do not, the longest is next to the
    contiguous run, so that taking the others apart makes the fewest parts."""
    dims: List[Tuple[int, int, int]] = []
    for y, x, n in sorted(((y, x, n) for n, x, y in zip(shape, strides, to_strides) if n != 1), reverse=True):
        if dims and dims[-1][1] == n * x and dims[-1][2] == n * y:
            dims[-1] = (dims[-1][0] * n, x, y)
        else:
            dims.append((n, x, y))
    run = [dims.pop()] if dims and dims[-1][1] == dims[-1][2] == 1 else []
    dims.sort(key=lambda d: d[0])
    return tuple(zip(*dims, *run)) or ((), (), ())


class _Reach(NamedTuple):
    """Where the elements of a tensor lie, from its address on, in bytes."""

    extent: int                          # from the first element's begin to the last one's end
    size: int                            # of an element
    steps: Tuple[Tuple[int, int], ...]   # (stride, extent) of the dimensions with more than one element


def _reach(shape: Tuple[int, ...], strides: Tuple[int, ...], size: int) -> _Reach:
    steps = tuple((s * size, n) for n, s in zip(shape, strides) if n > 1)
    return _Reach(0 if 0 in shape else size + sum(s * (n - 1) for s, n in steps), size, steps)


class _Layout(NamedTuple):
    """What states of one type, shape and strides and their results have in common."""

    beams_in: int
    to_shape: Tuple[int, ...]
    reach: _Reach
    to_reach: _Reach
    folded: bool    # whether elements of a result lie on each other, or might: their order in memory is not that of any order of the dimensions
    # (from_row, from_segment, to_row, to_segment, segments, bytes) and the segments' places in a state and in its result, in bytes
    launches: Tuple[Tuple[Tuple[int, ...], Tuple[Tuple[int, int], ...]], ...]


@functools.lru_cache(maxsize=256)
def _layout(shape: Tuple[int, ...], strides: Tuple[int, ...], to_strides: Tuple[int, ...], dtype: torch.dtype, items: int, beams_out: int) -> _Layout:
    if len(shape) < 1:
        raise ValueError("a state has the beams of all prompts along its first dimension, got a scalar")
    rows = int(shape[0])
    if items == 0 and rows or items and rows % items:
        raise ValueError(f"{rows} rows of a state {tuple(shape)} do not divide among {items} prompts")
    size = dtype.itemsize
    to_shape = (items * beams_out,) + tuple(shape[1:])
    row = strides[0] * size if rows > 1 else 0
    to_row = to_strides[0] * size if to_shape[0] > 1 else 0
    found: dict = {}
    if 0 not in to_shape:
        for at, to_at, n, nbytes, step, to_step in _segments(*_in_memory_order(shape[1:], strides[1:], to_strides[1:]), size):
            found.setdefault((row, step, to_row, to_step, n, nbytes), []).append((at, to_at))
    return _Layout(rows // items if items else 0, to_shape, _reach(shape, strides, size), _reach(to_shape, to_strides, size),
                   _folded(to_shape, to_strides), tuple((sizes, tuple(places)) for sizes, places in found.items()))


def _clusters(some: list, turn: int) -> List[list]:
    """The regions ``(begin, end, ...)`` that meet, directly or over others, in groups; on a circle of ``turn`` bytes, or a line where that is 0."""
    groups, end = [], 0
    for region in sorted(some):
        if groups and region[0] < end:
            groups[-1].append(region)
        else:
            groups.append([region])
        end = max(end, region[1])
    while turn and len(groups) > 1 and groups[0][0][0] < end - turn:  # the last one goes over the end and begins anew
        groups[-1] += groups.pop(0)
    return groups


def _clash(regions: list) -> bool:
    """Whether a result may share memory with another region; regions are ``(begin, end, reach, whether it is a result)`` in addresses.

    Ranges that do not meet share nothing.  Views of one buffer whose ranges interleave (keys and values side by side) are told apart by their addresses modulo
    a stride: where all longer strides of the regions are multiples of it, each occupies one interval there, as long as its shorter strides make it, and
    intervals that do not meet share nothing.  What no stride tells apart is taken to clash."""
    end = 0
    for region in sorted(regions):
        if region[0] < end:
            break
        end = region[1]
    else:
        return False

    def clash(some, moduli):
        if len(some) < 2 or not any(r[3] for r in some):
            return False
        for i, turn in enumerate(moduli):
            spans = {}
            for reach in {id(r[2]): r[2] for r in some}.values():  # few, of many regions
                span = reach.size + sum(s * (n - 1) for s, n in reach.steps if s < turn)
                if span > turn or any(s >= turn and s % turn for s, _ in reach.steps):
                    break
                spans[id(reach)] = span
            else:
                groups = _clusters([(r[0] % turn, r[0] % turn + spans[id(r[2])], r) for r in some], turn)
                if len(groups) > 1:
                    return any(clash([r for _, _, r in group], moduli[i + 1:]) for group in groups)
        return True

    return any(clash(group, sorted({s for reach in {id(r[2]): r[2] for r in group}.values() for s, _ in reach.steps if s > 0}, reverse=True)) for group in _clusters(regions, 0))


def beam_reorder(states: Sequence[torch.Tensor], parents: torch.Tensor, *, out: Optional[Sequence[torch.Tensor]] = None) -> List[torch.Tensor]:
    """Row ``n * B_out + j`` of each result is row ``n * B_in + parents[n, j]`` of its state, for states ``[N * B_in, ...]`` of any types and strides
    (the used part of a cache, say) and ``parents [N, B_out]`` int64; zeros where a parent lies outside ``[0, B_in)``.

    ``out``: tensors to write, of any strides (a state's own are the fastest); without it new contiguous ones.  ``out=states`` reorders in place (``B_out == B_in``, at most 128 beams): rows that keep their place
    are not moved.  A result is otherwise in memory of its own: one that may share an element with another result, with a state but the one that it is, or with
    ``parents`` is refused.  Views of one buffer that interleave without sharing an element are told apart.  Not differentiable, and no op that tracing sees: it
    works on addresses, so a compiled program is left for the call and goes on behind it."""
    states = list(states)
    if parents.dim() != 2:
        raise ValueError(f"expected parents [N, B], got {tuple(parents.shape)}")
    if parents.dtype != torch.int64:
        raise TypeError(f"parents must be int64, got {parents.dtype}")
    N, B_out = (int(x) for x in parents.shape)
    given = out is not None
    if given:
        results = list(out)
        if len(results) != len(states):
            raise ValueError(f"{len(results)} results for {len(states)} states")
    else:
        results = [t.new_empty((N * B_out,) + tuple(t.shape[1:])) for t in states]
    if not states:
        return results
    if torch.is_grad_enabled() and any([t.requires_grad for t in states + results]) or has_tangent(*states):
        raise ValueError("beam_reorder has no gradient: call it under torch.no_grad()")
    if True in [t.is_neg() for t in (states + results if given else states)]:
        raise ValueError(_NOT_ITS_VALUE)
    # What depends on the layout alone is looked at once for each: a model has many states and few layouts.
    kinds = list(zip([t.shape for t in states], [t.stride() for t in states], [u.stride() for u in results], [t.dtype for t in states]))
    groups = {kinds[0]: (states, results)}
    if kinds.count(kinds[0]) < len(kinds):
        groups = {}
        for kind, t, u in zip(kinds, states, results):
            some = groups.setdefault(kind, ([], []))
            some[0].append(t), some[1].append(u)
    used = []  # layouts with the addresses of each state and its result
    beams_in = -1
    for kind, (ts, us) in groups.items():
        layout = _layout(*kind, N, B_out)
        if beams_in not in (-1, layout.beams_in):
            raise ValueError(f"states of {beams_in} and of {layout.beams_in} beams a prompt")
        beams_in = layout.beams_in
        if given and ([u.shape for u in us].count(layout.to_shape) < len(us) or [u.dtype for u in us].count(kind[3]) < len(us)):
            raise ValueError(f"a result must be {layout.to_shape} {kind[3]}, got " + ", ".join(f"{tuple(u.shape)} {u.dtype}" for u in us))
        if kind[3].is_complex and any([t.is_conj() for t in ts + us]):
            raise ValueError(_NOT_ITS_VALUE)
        if given and layout.folded:
            raise ValueError("a result must not be expanded or overlap itself: its elements would be written more than once")
        if layout.to_reach.extent > 0:
            used.append((layout, kind[1] == kind[2] and beams_in == B_out, [t.data_ptr() for t in ts], [u.data_ptr() for u in us]))
    if not used:
        return results
    if given:
        regions = []
        for layout, may_be_same, ps, qs in used:
            reach, to_reach = layout.reach, layout.to_reach
            regions += [(q, q + to_reach.extent, to_reach, True) for q in qs]
            apart = [p for p, q in zip(ps, qs) if p != q] if may_be_same else ps
            if len(apart) < len(ps) and B_out > MAX_BEAMS:
                raise ValueError(f"at most {MAX_BEAMS} beams are reordered in place, got {B_out}")
            if reach.extent > 0:
                regions += [(p, p + reach.extent, reach, False) for p in apart]
        read = _reach(parents.shape, parents.stride(), 8)
        regions.append((parents.data_ptr(), parents.data_ptr() + read.extent, read, False))
        if _clash(regions):
            raise ValueError("a result shares memory with another result, with a state that it is not or with the parents, or may do so")
    device = parents.get_device()
    if device < 0 or [t.get_device() for t in states + results].count(device) < 2 * len(states):
        _require_device(parents, *states, *results)
    dev = _require_device(parents, states[0])
    if beams_in == 0:  # no row to take
        return [u.zero_() for u in results]
    lib, parents = _lib.load(), parents.contiguous()
    with device_guard(dev):
        stream = raw_stream(dev)
        for layout, _, ps, qs in used:
            pairs = list(zip(ps, qs))
            inside = [pair for pair in pairs if pair[0] == pair[1]]
            for some in (pairs,) if not inside or len(inside) == len(pairs) else (inside, [pair for pair in pairs if pair[0] != pair[1]]):
                for sizes, places in layout.launches:
                    every = [(p + x, q + y) for x, y in places for p, q in some] if places != ((0, 0),) else some
                    for at in range(0, len(every), _MAX_STATES):
                        from_, to = zip(*every[at:at + _MAX_STATES])
                        array = ctypes.c_void_p * len(from_)
                        st = lib.skyrl_logits_beam_reorder(array(*from_), array(*to), len(from_), *sizes, parents.data_ptr(), N, beams_in, B_out, stream)
                        _lib.check(st, "skyrl_logits_beam_reorder")
    if given:
        increment_version(results)
    return results
