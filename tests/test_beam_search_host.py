"""Host logic of beam search: workspace, refusals in front of any launch, layouts of states, shapes under fake tensors.  No GPU."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from skyrl_amd import _lib
from skyrl_amd import beam_search as BS

NULL, SHAPE, ALIGN, WORKSPACE, ARG = -1, -2, -3, -4, -5
P, BIG = 0x10000, 1 << 40


def test_workspace():
    size = _lib.load().skyrl_logits_beam_select_workspace_bytes
    assert size(1, 4, 1000, 8) == 4 * (16 + 8 * 8)       # short rows are not cut
    assert size(1, 4, 151936, 8) == 4 * 18 * (16 + 8 * 8)
    assert size(600, 1, 151936, 8) == 600 * (16 + 8 * 8)
    assert size(2, 3, 5, 15) == 6 * (16 + 5 * 8)
    for args in ((0, 4, 100, 2), (1, 0, 100, 2), (1, 129, 100, 2), (1, 4, 0, 2), (1, 4, 1 << 31, 2), (1, 4, 100, 0), (1, 4, 1000, 129), (1, 2, 3, 7), (BIG, 1, 100, 2),
                 (BIG, BIG, BIG, BIG), ((1 << 22) + 1, 1, 100, 2)):
        assert size(*args) == 0


def test_selection_arguments_are_checked_before_a_launch():
    def select(logits=P, dtype=0, ld_item=400, ld_beam=100, scores=P, items=2, beams=4, V=100, k=3, rcp=1.0, out=P, parents=P, tokens=P, ws=P, nbytes=BIG):
        return _lib.load().skyrl_logits_beam_select(logits, dtype, ld_item, ld_beam, scores, items, beams, V, k, rcp, out, parents, tokens, ws, nbytes, None)

    assert [select(logits=None), select(scores=None), select(out=None), select(parents=None), select(tokens=None), select(dtype=3), select(items=0), select(beams=129),
            select(V=0), select(k=0), select(k=129, V=1000), select(k=9, V=2), select(ld_item=-1), select(ld_beam=BIG), select(logits=P + 1),
            select(dtype=1, logits=P + 2), select(scores=P + 2), select(tokens=P + 4), select(ws=P + 4), select(rcp=0.0), select(rcp=math.nan), select(rcp=1e39),
            select(rcp=-1.0), select(rcp=1e-300), select(ws=None), select(nbytes=64)] == \
        [NULL] * 5 + [ARG] + [SHAPE] * 8 + [ALIGN] * 5 + [ARG] * 5 + [WORKSPACE] * 2


def test_reordering_arguments_are_checked_before_a_launch():
    def reorder(src=(P,), dst=(2 * P,), count=None, from_row=64, from_segment=16, to_row=64, to_segment=16, segments=4, nbytes=16, parents=P, items=1, beams_in=2,
                beams_out=3):
        a = None if src is None else (ctypes.c_void_p * max(1, len(src)))(*src)
        b = None if dst is None else (ctypes.c_void_p * max(1, len(dst)))(*dst)
        return _lib.load().skyrl_logits_beam_reorder(a, b, len(src or ()) if count is None else count, from_row, from_segment, to_row, to_segment, segments, nbytes,
                                                     parents, items, beams_in, beams_out, None)

    assert [reorder(src=None, count=1), reorder(dst=None), reorder(parents=None), reorder(src=(None,)), reorder(count=0), reorder(count=201), reorder(segments=0),
            reorder(nbytes=0), reorder(items=0), reorder(beams_in=0), reorder(beams_out=0), reorder(items=1 << 20, beams_out=1 << 20), reorder(from_row=-1),
            reorder(to_segment=BIG), reorder(items=1 << 30), reorder(nbytes=(1 << 35) + 1, segments=1), reorder(parents=P + 4), reorder(dst=(P,)),
            reorder(dst=(P,), beams_out=2, to_row=128), reorder(dst=(P,), beams_in=129, beams_out=129), reorder(src=(P, P), dst=(2 * P, P)),
            reorder(src=(P, 3 * P), dst=(P, 5 * P), beams_out=2)] == \
        [NULL] * 4 + [SHAPE] * 12 + [ALIGN] + [ARG] * 5


def test_refusals():
    z, s = torch.zeros(2, 3, 50), torch.zeros(2, 3)
    with pytest.raises(RuntimeError):  # no CPU implementation
        BS.beam_select(z, s, 2)
    for logits, scores, k in ((z[0], s, 2), (z, s[:, :2], 2), (z, s, 0), (z, s, 129), (z[:, :, :1], s, 4), (torch.zeros(1, 129, 4), torch.zeros(1, 129), 2),
                              (z[:, :0], s[:, :0], 1), (z.requires_grad_(), s, 2), (z.detach(), s.clone().requires_grad_(), 2)):
        with pytest.raises(ValueError):
            BS.beam_select(logits, scores, k)
    z = z.detach()
    for logits, scores in ((z.half(), s), (z, s.double())):
        with pytest.raises(TypeError):
            BS.beam_select(logits, scores, 2)
    for temperature in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            BS.beam_select(z, s, 2, temperature=temperature)
    t, p = torch.zeros(6, 4), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(RuntimeError):
        BS.beam_reorder([t], p)
    with pytest.raises(TypeError):
        BS.beam_reorder([t], p.int())
    for states, parents, out in (([t], p[0], None), ([t[:5]], p, None), ([t, t[:4]], p, None), ([torch.zeros(())], p, None), ([t], p, []), ([t], p, [t[:4]]),
                                 ([t], p, [t.double()]), ([t], p, [torch.zeros(6, 1).expand(6, 4)]), ([t], p[:0], None), ([t.clone().requires_grad_()], p, None)):
        with pytest.raises(ValueError):
            BS.beam_reorder(states, parents, out=out)


def test_nothing_to_do():
    assert BS.beam_reorder([], torch.zeros(2, 3, dtype=torch.int64)) == []
    (t,) = BS.beam_reorder([torch.zeros(6, 0, 4)], torch.zeros(2, 5, dtype=torch.int64))
    assert t.shape == (10, 0, 4)


@pytest.mark.parametrize("state,want", [
    (torch.empty(6, 2, 40, 64)[:, :, :33], (2, 33 * 64 * 4, 40 * 64 * 4)), (torch.empty(6, 5, 7), (1, 140, 0)), (torch.empty(6), (1, 4, 0)),
    (torch.empty(6, 3)[:, :1], (1, 4, 0)), (torch.empty(6, 9, 10).transpose(1, 2), None), (torch.empty(6, 8, 3)[:, ::2], (4, 12, 24)),
])
def test_segments_of_a_row(state, want):
    got = BS._segments(tuple(state.shape[1:]), state.stride()[1:], state.stride()[1:], 4)
    if want is None:  # columns that do not join: one element at a time, along the last dimension
        assert sum(n * b for _, _, n, b, _, _ in got) == state[0].numel() * 4
        assert sorted(at + i * step for at, _, n, b, step, _ in got for i in range(n)) == list(range(0, state[0].numel() * 4, 4))
    else:
        assert [(n, b, step) for _, _, n, b, step, _ in got] == [want] and got[0][4] == got[0][5]


def test_shapes_under_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        r = BS.beam_select(torch.empty(2, 3, 50, dtype=torch.bfloat16), torch.empty(2, 3), 7)
        assert r.scores.shape == r.parents.shape == r.tokens.shape == (2, 7) and r.tokens.dtype == torch.int64 and r.scores.dtype == torch.float32


def test_views_whose_memory_is_not_their_value_are_refused():
    c = torch.zeros(6, 4, dtype=torch.complex64)
    p = torch.zeros(2, 3, dtype=torch.int64)
    for state in (c.conj(), c.conj().imag):
        with pytest.raises(ValueError):
            BS.beam_reorder([state], p)
        with pytest.raises(ValueError):
            BS.beam_reorder([torch.zeros_like(state)], p, out=[state])


@pytest.mark.parametrize("size,stride,refused", [((6, 4), (4, 1), False), ((6, 4), (1, 6), False), ((6, 2, 5), (40, 20, 2), False), ((6, 4), (3, 1), True),
                                                 ((6, 4), (1, 1), True), ((6, 4), (4, 0), True), ((6, 1), (1, 0), False)])
def test_results_that_overlap_themselves_are_refused(size, stride, refused):
    t = torch.zeros(300).as_strided(size, stride)
    p = torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(ValueError if refused else RuntimeError) as e:  # RuntimeError: not on a GPU
        BS.beam_reorder([torch.zeros(size)], p, out=[t])
    assert ("overlap" in str(e.value)) == refused
