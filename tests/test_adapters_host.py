"""Host logic of the head with adapters and of the best alternatives: workspace queries, refusals in front of any launch, shapes under fake
tensors.  No GPU."""

from __future__ import annotations

import itertools
import math

import pytest
import torch

from skyrl_amd import _lib
from skyrl_amd import adapters as AD
from skyrl_amd import torch_utils as TU

NULL, SHAPE, ALIGN, WORKSPACE, ARG = -1, -2, -3, -4, -5
P = 0x10000


def test_workspaces():
    lib = _lib.load()
    rows = lambda T, Rp: 4 * (T + 1) * Rp + 4 * T  # noqa: E731
    assert rows(300, 32) <= lib.skyrl_lmhead_adapter_logits_workspace_bytes(300, 896, 1, 24) <= rows(300, 32) + 1024
    grouped = rows(300, 32) + 300 * (8 + 4 + 2 * 896)   # rows of several adapters are brought together
    assert grouped <= lib.skyrl_lmhead_adapter_logits_workspace_bytes(300, 896, 5, 24) <= grouped + 2048
    head = lib.skyrl_lmhead_fwd_workspace_bytes(300, 896, 5000)
    assert head + rows(300, 64) <= lib.skyrl_lmhead_adapter_fwd_workspace_bytes(300, 896, 5000, 1, 64) <= head + rows(300, 64) + 1024
    small, large = (lib.skyrl_lmhead_adapter_bwd_workspace_bytes(300, 896, 5000, n, 16) for n in (1, 64))
    assert lib.skyrl_lmhead_bwd_active_rows_workspace_bytes(300, 896, 5000, 0) < small < large
    # what does not fit any call has no workspace
    for T, H, V, N, R in ((0, 64, 8, 1, 8), (8, 64, 0, 1, 8), (8, 64, 8, 0, 8), (8, 64, 8, 65536, 8), (8, 64, 8, 1, 257), (1 << 31, 64, 8, 1, 8)):
        assert lib.skyrl_lmhead_adapter_bwd_workspace_bytes(T, H, V, N, R) == 0
    for T, R in ((0, 8), (1 << 40, 8), (8, 0), (8, 264)):
        assert lib.skyrl_lmhead_adapter_logits_workspace_bytes(T, 64, 1, R) == 0
    big = (1, 300, 1 << 20, (1 << 31) - 1, 1 << 40)
    for T, V, N in itertools.product(big, (5, 152064, 1 << 40), (1, 65535, 1 << 40)):
        lib.skyrl_lmhead_adapter_bwd_workspace_bytes(T, 3584, V, N, 256)


def adapter_args(a=P, a_adapter=16 * 64, a_row=64, b=P, b_adapter=16 * 100, b_row=16, scaling=P, ids=P, N=2, R=16):
    return a, a_adapter, a_row, b, b_adapter, b_row, scaling, ids, N, R


BAD_ADAPTERS = [(dict(a=None), NULL), (dict(b=None), NULL), (dict(scaling=None), NULL), (dict(ids=None), NULL), (dict(N=0), SHAPE), (dict(N=65536), SHAPE),
                (dict(R=12), SHAPE), (dict(R=0), SHAPE), (dict(R=264), SHAPE), (dict(a_row=56), SHAPE), (dict(b_row=8), SHAPE),
                (dict(a_adapter=-8), SHAPE), (dict(b_adapter=1 << 41), SHAPE), (dict(a=P + 8), ALIGN), (dict(b=P + 2), ALIGN), (dict(a_row=68), ALIGN),
                (dict(b_row=20), ALIGN), (dict(a_adapter=1028), ALIGN), (dict(scaling=P + 2), ALIGN), (dict(ids=P + 4), ALIGN)]


@pytest.mark.parametrize("bad,status", BAD_ADAPTERS)
def test_adapters_are_checked_before_a_launch(bad, status):
    lib = _lib.load()
    ad = adapter_args(**bad)
    big = 1 << 40
    assert lib.skyrl_lmhead_adapter_fwd(P, 64, P, 64, P, *ad, 8, 64, 100, 1.0, P, P, P, P, P, big, None) == status
    assert lib.skyrl_lmhead_adapter_logits(P, 64, P, 64, *ad, 8, 64, 100, 0, P, 100, P, big, None) == status
    assert lib.skyrl_lmhead_adapter_bwd(P, 64, P, 64, P, *ad, P, P, P, None, 8, 64, 100, 1.0, P, P, P, P, big, None) == status


def test_other_arguments_are_checked_before_a_launch():
    lib = _lib.load()
    ad, big = adapter_args(), 1 << 40

    def fwd(hidden=P, ldh=64, labels=P, T=8, H=64, V=100, rcp=1.0, lp=P, ws=P, nbytes=big):
        return lib.skyrl_lmhead_adapter_fwd(hidden, ldh, P, 64, labels, *ad, T, H, V, rcp, lp, P, P, P, ws, nbytes, None)

    assert [fwd(hidden=None), fwd(ldh=63), fwd(labels=None), fwd(T=0), fwd(H=60), fwd(V=0), fwd(rcp=0.0), fwd(rcp=math.inf), fwd(lp=None), fwd(ws=None),
            fwd(nbytes=1024), fwd(ws=P + 64)] == [NULL, SHAPE, NULL, SHAPE, SHAPE, SHAPE, ARG, ARG, NULL, WORKSPACE, WORKSPACE, ALIGN]

    def logits(dtype=0, out=P, ld=100, ws=P, nbytes=big):
        return lib.skyrl_lmhead_adapter_logits(P, 64, P, 64, *ad, 8, 64, 100, dtype, out, ld, ws, nbytes, None)

    assert [logits(dtype=2), logits(out=None), logits(out=P + 1), logits(dtype=1, out=P + 2), logits(ld=99), logits(ws=None), logits(nbytes=64),
            logits(ws=P + 128)] == [ARG, NULL, ALIGN, ALIGN, SHAPE, WORKSPACE, WORKSPACE, ALIGN]

    def bwd(lse=P, pz=None, g=P, q=None, dh=P, da=P, db=P, ws=P, nbytes=big):
        return lib.skyrl_lmhead_adapter_bwd(P, 64, P, 64, P, *ad, lse, pz, g, q, 8, 64, 100, 1.0, dh, da, db, ws, nbytes, None)

    assert [bwd(lse=None), bwd(g=None), bwd(q=P), bwd(dh=None), bwd(da=None), bwd(db=None), bwd(da=P + 8), bwd(ws=None), bwd(nbytes=1 << 16)] == \
        [NULL, NULL, NULL, NULL, NULL, NULL, ALIGN, WORKSPACE, WORKSPACE]


def test_top_arguments_are_checked_before_a_launch():
    lib = _lib.load()

    def fwd(logits=P, dtype=1, ld=64, labels=P, T=4, V=64, k=2, rcp=1.0, ranks=P, top=P, top_ids=P, ws=None, nbytes=0):
        return lib.skyrl_logits_top_fwd(logits, dtype, ld, labels, T, V, k, rcp, None, None, None, None, ranks, top, top_ids, ws, nbytes, None)

    assert [fwd(logits=None), fwd(dtype=2), fwd(ld=63), fwd(labels=None), fwd(T=0), fwd(V=0), fwd(k=65), fwd(k=-1), fwd(V=1 << 31, ld=1 << 31),
            fwd(rcp=0.0), fwd(rcp=math.nan), fwd(top=None), fwd(top_ids=None), fwd(top_ids=P + 4), fwd(logits=P + 2)] == \
        [NULL, ARG, SHAPE, NULL, SHAPE, SHAPE, SHAPE, SHAPE, SHAPE, ARG, ARG, NULL, NULL, ALIGN, ALIGN]
    need = lib.skyrl_logits_top_workspace_bytes(4, 152064, 20)
    assert 4 * 18 * 20 * 8 < need < 4 * 64 * 20 * 8 and lib.skyrl_logits_top_workspace_bytes(4096, 152064, 20) == 0
    assert [fwd(ld=152064, V=152064, k=20), fwd(ld=152064, V=152064, k=20, ws=P, nbytes=need - 1), fwd(ld=152064, V=152064, k=20, ws=P + 4, nbytes=need)] == \
        [WORKSPACE, WORKSPACE, ALIGN]
    for T, V, k in ((0, 64, 2), (4, 0, 0), (4, 64, 65), (4, 64, 129), (1 << 40, 64, 2), (4, 1 << 40, 2)):
        assert lib.skyrl_logits_top_workspace_bytes(T, V, k) == 0

    def bwd(lse=P, pz=P, g=P, q=None, top_ids=P, dtop=P, k=2, out=P + 4096, ldd=64, labels=P):
        return lib.skyrl_logits_top_bwd(P, 1, 64, labels, lse, pz, g, q, top_ids, dtop, 4, 64, k, 1.0, out, ldd, None)

    assert [bwd(lse=None), bwd(g=None, dtop=None), bwd(q=P, pz=None), bwd(top_ids=None), bwd(out=None), bwd(ldd=63), bwd(k=129), bwd(out=P + 256),
            bwd(labels=None), bwd(out=P + 2)] == [NULL, NULL, NULL, NULL, NULL, SHAPE, SHAPE, ARG, NULL, ALIGN]


def test_shapes_under_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        h, w = torch.empty(6, 64, dtype=torch.bfloat16), torch.empty(100, 64, dtype=torch.bfloat16)
        a, b = torch.empty(3, 8, 64, dtype=torch.bfloat16), torch.empty(3, 100, 8, dtype=torch.bfloat16)
        s, ids, y = torch.empty(3), torch.empty(6, dtype=torch.int64), torch.empty(6, dtype=torch.int64)
        z = AD.adapter_logits(h, w, a, b, s, ids, dtype=torch.float32)
        assert z.shape == (6, 100) and z.dtype == torch.float32
        r = TU.top_logprobs_from_logits(z, y, 7)
        assert r.top_ids.shape == (6, 7) and r.ranks.dtype == torch.int64 and r.logprobs.shape == (6,)
        lp, ent = AD.adapter_logprobs_from_hidden(h, w, y, a.requires_grad_(), b.requires_grad_(), s, ids)
        lp.sum().backward()
        assert a.grad.shape == a.shape and b.grad.shape == b.shape


def test_cpu_tensors_are_refused():
    z, y = torch.zeros(2, 50), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError):
        TU.top_logprobs_from_logits(z, y, 2)
    h, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(50, 64, dtype=torch.bfloat16)
    a, b = torch.zeros(1, 8, 64, dtype=torch.bfloat16), torch.zeros(1, 50, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        AD.adapter_logits(h, w, a, b, torch.ones(1), y)


def test_stack_adapters():
    pairs = [(torch.ones(r, 64), torch.ones(30, r)) for r in (4, 16, 1)]
    a, b, s = AD.stack_adapters(pairs, [1, 2, 3])
    assert a.shape == (3, 16, 64) and b.shape == (3, 30, 16) and a.dtype == torch.bfloat16 and s.tolist() == [1.0, 2.0, 3.0]
    assert float(a[0].sum()) == 4 * 64 and float(b[2].sum()) == 30
    for bad in ([(torch.ones(4, 64), torch.ones(30, 5))], [(torch.ones(4, 64), torch.ones(30, 4)), (torch.ones(4, 32), torch.ones(30, 4))]):
        with pytest.raises(ValueError):
            AD.stack_adapters(bad, [1.0] * len(bad))
