"""Which way ``top_logprobs_from_logits`` takes: past the registered op only where nothing can tell the difference.  On the CPU, with a function in
the kernels' place that reads what lies at the tensors' addresses, as a kernel does."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from skyrl_amd import torch_utils as TU

T, V, K = 3, 7, 2


def at_address(t: torch.Tensor, c_type) -> torch.Tensor:
    t = t.contiguous()  # the dispatcher expands a zero tensor from one element
    if t.data_ptr() == 0:
        raise RuntimeError("a kernel would read from address 0")
    return torch.frombuffer((c_type * t.numel()).from_address(t.data_ptr()), dtype=t.dtype).reshape(t.shape).clone()


@pytest.fixture
def taken(monkeypatch):
    """The calls of the function: whether they wanted what only a backward reads (the op) or not (the way past it)."""
    calls = []

    def read(logits, labels, k, rcp_temperature, want_rows):
        calls.append(want_rows)
        z = at_address(logits, ctypes.c_float).double() * rcp_temperature
        y = at_address(labels, ctypes.c_int64)
        lsm = torch.log_softmax(z, 1)
        lp = lsm.gather(1, y[:, None])[:, 0].float()
        top = lsm.topk(k, 1)
        rows = (torch.zeros(T), torch.zeros(T)) if want_rows else (None, None)
        return (lp, -(lsm.exp() * lsm).sum(1).float(), *rows, 1 + (lsm > lsm.gather(1, y[:, None])).sum(1), top.values.float(), top.indices)

    monkeypatch.setattr(TU, "_top_fwd", read)
    return calls


def inputs():
    gen = torch.Generator().manual_seed(1)
    return torch.randn(T, V, generator=gen), torch.randint(0, V, (T,), generator=gen)


def expect(got, z, y):
    lsm = torch.log_softmax(z.double(), 1)
    assert torch.allclose(got.logprobs.double(), lsm.gather(1, y[:, None])[:, 0], atol=1e-6)
    assert torch.equal(got.top_ids, lsm.topk(K, 1).indices)


def test_a_plain_call_goes_past_the_op(taken):
    z, y = inputs()
    expect(TU.top_logprobs_from_logits(z, y, K), z, y)
    with torch.no_grad():
        expect(TU.top_logprobs_from_logits(z.clone().requires_grad_(), y, K), z, y)
    assert taken == [False, False]


def test_tensors_whose_memory_is_not_their_value(taken):
    z, y = inputs()
    expect(TU.top_logprobs_from_logits(torch._neg_view(z), y, K), -z, y)
    expect(TU.top_logprobs_from_logits(z, torch._neg_view(-y), K), z, y)
    zeros = TU.top_logprobs_from_logits(torch._efficientzerotensor(T, V), y, K)
    assert torch.allclose(zeros.logprobs, torch.log_softmax(torch.zeros(V), 0)[0].expand(T))
    assert all(taken)
    imaginary = torch.complex(torch.zeros_like(z), z).conj().imag  # every other element: a copy, whose memory is its value
    expect(TU.top_logprobs_from_logits(imaginary, y, K), -z, y)


def test_tensors_without_memory_give_shapes(taken):
    z, y = inputs()
    r = TU.top_logprobs_from_logits(z.to("meta"), y.to("meta"), K)
    assert r.logprobs.is_meta and r.top_ids.shape == (T, K) and r.ranks.dtype == torch.int64 and not taken


def test_a_tangent_is_not_dropped(taken):
    z, y = inputs()
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward"):
            TU.top_logprobs_from_logits(forward_ad.make_dual(z, torch.ones_like(z)), y, K)
        expect(TU.top_logprobs_from_logits(z, y, K), z, y)  # a level alone changes nothing
    assert taken[-1] is False


def test_a_gradient_is_recorded(taken):
    z, y = inputs()
    r = TU.top_logprobs_from_logits(z.requires_grad_(), y, K)
    assert r.logprobs.requires_grad and r.top_logprobs.requires_grad and not r.ranks.requires_grad and taken == [True]
