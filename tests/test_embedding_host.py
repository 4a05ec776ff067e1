"""Host logic of the embedding: workspace, refusals in front of any launch, shapes under fake tensors.  No GPU."""

from __future__ import annotations

import math

import pytest
import torch

from skyrl_amd import _lib
from skyrl_amd import embedding as E

NULL, SHAPE, ALIGN, WORKSPACE, ARG = -1, -2, -3, -4, -5
P, BIG = 0x10000, 1 << 40


def test_workspace():
    lib = _lib.load()
    size = lib.skyrl_lmhead_embedding_bwd_workspace_bytes
    assert 8 <= size(1, 64, 100) <= 1024
    # sorted ids, and two fp32 rows for each sixteen tokens; twice the ids where blocks are merged
    assert 300 * 8 + 19 * 2 * 64 * 4 <= size(300, 64, 100) <= 300 * 8 + 19 * 2 * 64 * 4 + 1024
    assert 5000 * 16 + 313 * 2 * 64 * 4 <= size(5000, 64, 100) <= 5000 * 16 + 313 * 2 * 64 * 4 + 2048
    for T, H, V in ((0, 64, 8), (8, 0, 8), (8, 64, 0), ((1 << 24) + 1, 64, 8), (8, (1 << 22) + 1, 8), (8, 64, (1 << 31) - 1), (1 << 24, 1 << 16, 8),
                    (-1, 64, 8), (1 << 62, 1 << 62, 1 << 62)):
        assert size(T, H, V) == 0
    assert size(1 << 24, 1 << 10, 152064) > 0


def test_forward_arguments_are_checked_before_a_launch():
    def fwd(table=P, dtype=0, ld=64, ids=P, T=4, H=64, V=100, scale=1.0, out=P):
        return _lib.load().skyrl_lmhead_embedding_fwd(table, dtype, ld, ids, T, H, V, scale, out, None)

    assert [fwd(table=None), fwd(ids=None), fwd(out=None), fwd(dtype=2), fwd(T=0), fwd(H=0), fwd(V=0), fwd(T=BIG), fwd(H=BIG, ld=BIG), fwd(V=BIG), fwd(ld=63),
            fwd(ld=BIG), fwd(table=P + 1), fwd(out=P + 1), fwd(dtype=1, out=P + 2), fwd(ids=P + 4), fwd(scale=math.nan), fwd(scale=math.inf)] == \
        [NULL, NULL, NULL, ARG, SHAPE, SHAPE, SHAPE, SHAPE, SHAPE, SHAPE, SHAPE, SHAPE, ALIGN, ALIGN, ALIGN, ALIGN, ARG, ARG]


def test_backward_arguments_are_checked_before_a_launch():
    def bwd(dout=P, dtype=0, ld=64, ids=P, T=40, H=64, V=100, scale=1.0, add=0, out=P, ws=P, nbytes=BIG):
        return _lib.load().skyrl_lmhead_embedding_bwd(dout, dtype, ld, ids, -1, T, H, V, scale, add, out, ws, nbytes, None)

    assert [bwd(dout=None), bwd(ids=None), bwd(out=None), bwd(dtype=-1), bwd(T=0), bwd(T=BIG), bwd(H=0), bwd(V=0), bwd(V=BIG), bwd(ld=63), bwd(ld=-64),
            bwd(T=1 << 24, H=1 << 16, ld=1 << 16), bwd(dout=P + 1), bwd(out=P + 1), bwd(add=1, out=P + 2), bwd(ids=P + 4), bwd(scale=-math.inf), bwd(add=2),
            bwd(ws=None), bwd(nbytes=1024), bwd(ws=P + 128)] == \
        [NULL, NULL, NULL, ARG, SHAPE, SHAPE, SHAPE, SHAPE, SHAPE, SHAPE, SHAPE, SHAPE, ALIGN, ALIGN, ALIGN, ALIGN, ARG, ARG, WORKSPACE, WORKSPACE, ALIGN]


def test_refusals():
    w, ids = torch.zeros(10, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError):  # no CPU implementation
        E.embedding_lookup(w, ids)
    for bad in (w.double(), w.half(), w[0]):
        with pytest.raises(TypeError):
            E.embedding_lookup(bad, ids)
    with pytest.raises(ValueError):
        E.embedding_lookup(w.t(), ids)
    for bad in (ids.float(), ids.bool(), ids.to(torch.int16)):
        with pytest.raises(TypeError):
            E.embedding_lookup(w, bad)
    for scale in (math.nan, math.inf, 1e39):
        with pytest.raises(ValueError):
            E.embedding_lookup(w, ids, scale=scale)
    for padding in (10, -11):
        with pytest.raises(ValueError):
            E.embedding_lookup(w, ids, padding_idx=padding)
    d = torch.zeros(3, 8)
    for buffer in (w.to(torch.bfloat16), w[:, :4], w[0]):
        with pytest.raises(ValueError):
            E.embedding_backward_accumulate(d, ids, buffer)
    for grad, tokens in ((d[:2], ids), (torch.zeros(3, 4), ids), (d, ids[:2])):
        with pytest.raises(ValueError):
            E.embedding_backward_accumulate(grad, tokens, w)
    with pytest.raises(ValueError):
        E.embedding_backward_accumulate(d, ids, w.clone().requires_grad_())
    with pytest.raises(TypeError):
        E.embedding_backward_accumulate(d.double(), ids, w)


def test_shapes_under_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        w = torch.empty(100, 24, dtype=torch.bfloat16).requires_grad_()
        out = E.embedding_lookup(w, torch.empty(2, 5, dtype=torch.int32), scale=3.0, padding_idx=-1)
        assert out.shape == (2, 5, 24) and out.dtype == torch.bfloat16
        out.sum().backward()
        assert w.grad.shape == w.shape and w.grad.dtype == w.dtype
