"""Host logic of the head in 8-bit integers: workspaces, refusals in front of any launch, shapes under fake tensors.  No GPU."""

from __future__ import annotations

import math

import pytest
import torch

from skyrl_amd import _lib
from skyrl_amd import int8_head as I

NULL, SHAPE, ALIGN, WORKSPACE, ARG = -1, -2, -3, -4, -5
P, BIG = 0x10000, 1 << 40


def test_workspaces():
    lib = _lib.load()
    assert 300 * 896 + 300 * 4 <= lib.skyrl_lmhead_int8_logits_workspace_bytes(300, 896) <= 300 * 900 + 1024
    assert 300 * 256 + 300 * 4 <= lib.skyrl_lmhead_int8_logits_workspace_bytes(300, 129) <= 300 * 260 + 1024
    head = lib.skyrl_lmhead_fwd_workspace_bytes(300, 896, 5000)
    assert head + 300 * 900 <= lib.skyrl_lmhead_int8_fwd_workspace_bytes(300, 896, 5000) <= head + 300 * 900 + 2048
    # of a block of tokens, however many there are
    assert lib.skyrl_lmhead_int8_fwd_workspace_bytes(1 << 30, 896, 5000) == lib.skyrl_lmhead_int8_fwd_workspace_bytes(32768, 896, 5000)
    for T, H, V in ((0, 64, 8), (8, 0, 8), (8, 64, 0), (8, 132097, 8), ((1 << 30) + 1, 64, 8), (8, 64, 1 << 31), (BIG, BIG, BIG)):
        assert lib.skyrl_lmhead_int8_fwd_workspace_bytes(T, H, V) == 0
    assert lib.skyrl_lmhead_int8_logits_workspace_bytes(8, 132096) > 0 == lib.skyrl_lmhead_int8_logits_workspace_bytes(8, 132097)


BAD = [(dict(hidden=None), NULL), (dict(values=None), NULL), (dict(scale=None), NULL), (dict(dtype=2), ARG), (dict(dtype=-1), ARG), (dict(T=0), SHAPE),
       (dict(H=0), SHAPE), (dict(ld=99), SHAPE), (dict(ld=BIG), SHAPE), (dict(ldv=112), SHAPE), (dict(H=132097, ld=BIG - 1, ldv=1 << 20), SHAPE),
       (dict(ldv=(1 << 23) + 16), SHAPE), (dict(T=BIG), SHAPE), (dict(hidden=P + 1), ALIGN), (dict(dtype=1, hidden=P + 2), ALIGN), (dict(values=P + 8), ALIGN),
       (dict(ldv=136), ALIGN), (dict(scale=P + 2), ALIGN)]


@pytest.mark.parametrize("bad,status", BAD)
def test_operands_are_checked_before_a_launch(bad, status):
    lib = _lib.load()
    a = {**dict(hidden=P, dtype=0, ld=100, values=P, ldv=128, scale=P, T=8, H=100), **bad}
    lead = (a["hidden"], a["dtype"], a["ld"])
    assert lib.skyrl_lmhead_int8_rows(*lead, a["T"], a["H"], a["values"], a["ldv"], a["scale"], None) == status
    head = (a["values"], a["ldv"], a["scale"])
    assert lib.skyrl_lmhead_int8_fwd(*lead, *head, P, a["T"], a["H"], 50, 1.0, P, P, P, BIG, None) == status
    assert lib.skyrl_lmhead_int8_logits(*lead, *head, a["T"], a["H"], 50, 0, P, 50, P, BIG, None) == status


def test_other_arguments_are_checked_before_a_launch():
    lib = _lib.load()

    def fwd(labels=P, V=50, rcp=1.0, lp=P, ws=P, nbytes=BIG):
        return lib.skyrl_lmhead_int8_fwd(P, 0, 100, P, 128, P, labels, 8, 100, V, rcp, lp, None, ws, nbytes, None)

    assert [fwd(labels=None), fwd(lp=None), fwd(V=0), fwd(V=BIG), fwd(labels=P + 4), fwd(rcp=0.0), fwd(rcp=math.inf), fwd(rcp=math.nan), fwd(ws=None),
            fwd(nbytes=1024), fwd(ws=P + 64)] == [NULL, NULL, SHAPE, SHAPE, ALIGN, ARG, ARG, ARG, WORKSPACE, WORKSPACE, ALIGN]

    def logits(dtype=0, out=P, ld=50, ws=P, nbytes=BIG):
        return lib.skyrl_lmhead_int8_logits(P, 0, 100, P, 128, P, 8, 100, 50, dtype, out, ld, ws, nbytes, None)

    assert [logits(dtype=2), logits(out=None), logits(out=P + 1), logits(dtype=1, out=P + 2), logits(ld=49), logits(ld=BIG), logits(ws=None), logits(nbytes=64),
            logits(ws=P + 128)] == [ARG, NULL, ALIGN, ALIGN, SHAPE, SHAPE, WORKSPACE, WORKSPACE, ALIGN]
    assert lib.skyrl_lmhead_int8_rows(P, 0, 100, (1 << 23) + 1, 100, P, 128, P, None) == SHAPE


def test_refusals():
    h, y = torch.zeros(2, 64), torch.zeros(2, dtype=torch.int64)
    head = I.Int8Head(torch.zeros(50, 128, dtype=torch.int8), torch.zeros(50))
    for call in (lambda: I.int8_logits(h, head), lambda: I.int8_logprobs_from_hidden(h, head, y), lambda: I.quantize_head(torch.zeros(5, 64))):
        with pytest.raises(RuntimeError):  # no CPU implementation
            call()
    for bad in (I.Int8Head(head.values[:, :64], head.scale), I.Int8Head(head.values, head.scale[:9]), I.Int8Head(torch.zeros(50, 256, dtype=torch.int8), head.scale),
                I.Int8Head(head.values[:0], head.scale[:0]), I.Int8Head(torch.zeros(128, 50, dtype=torch.int8).t(), head.scale),
                I.Int8Head(head.values, torch.zeros(100)[::2])):
        with pytest.raises(ValueError):
            I.int8_logits(h, bad)
        with pytest.raises(ValueError):
            I.int8_logprobs_from_hidden(h, bad, y)
    for bad in (I.Int8Head(head.values.to(torch.uint8), head.scale), I.Int8Head(head.values, head.scale.double())):
        with pytest.raises(TypeError):
            I.int8_logits(h, bad)
    for bad in (h.half(), h.double()):
        with pytest.raises(TypeError):
            I.int8_logits(bad, head)
    with pytest.raises(TypeError):
        I.int8_logits(h, head, dtype=torch.float16)
    with pytest.raises(ValueError):
        I.int8_logits(torch.zeros(2, 0), head)
    with pytest.raises(ValueError):
        I.int8_logits(h.clone().requires_grad_(), head)
    with pytest.raises(ValueError):
        I.int8_logprobs_from_hidden(h, I.Int8Head(head.values, torch.zeros(50, requires_grad=True)), y)
    for labels in (y[:1], torch.zeros(2, 1, dtype=torch.int64)):
        with pytest.raises(ValueError):
            I.int8_logprobs_from_hidden(h, head, labels)
    with pytest.raises(TypeError):
        I.int8_logprobs_from_hidden(h, head, y.float())
    for temperature in (0.0, -1.0, math.nan, math.inf, 1e-39):
        with pytest.raises(ValueError):
            I.int8_logprobs_from_hidden(h, head, y, temperature=temperature)
    with pytest.raises(TypeError):
        I.quantize_head(torch.zeros(5, 64, dtype=torch.float16))
    with pytest.raises(ValueError):
        I.quantize_head(torch.zeros(5, 132097))


def test_shapes_under_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        head = I.quantize_head(torch.empty(100, 200, dtype=torch.bfloat16))
        assert head.values.shape == (100, 256) and head.values.dtype == torch.int8 and head.scale.shape == (100,)
        h = torch.empty(2, 3, 200)
        assert I.int8_logits(h, head, dtype=torch.float32).shape == (2, 3, 100)
        lp, ent = I.int8_logprobs_from_hidden(h, head, torch.empty(2, 3, dtype=torch.int64))
        assert lp.shape == ent.shape == (2, 3) and lp.dtype == torch.float32
