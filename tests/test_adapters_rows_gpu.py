"""Hidden states whose rows lie in ways that the kernels do not walk: they are copied, and nothing else changes."""

from __future__ import annotations

import pytest
import torch

from skyrl_amd import adapters as AD
from test_adapters_gpu import make, on


def pitched(hidden, pitch):
    """The same rows, `pitch` elements apart."""
    wide = torch.full((hidden.shape[0], pitch), 7.0, dtype=hidden.dtype, device=hidden.device)
    wide[:, :hidden.shape[1]] = hidden
    return wide[:, :hidden.shape[1]]


@pytest.mark.parametrize("pitch", [64, 65, 66, 68, 72, 100])
def test_rows_that_do_not_begin_on_16_bytes_are_copied(pitch):
    hidden = torch.randn(5, 64).to(torch.bfloat16)
    rows, ids = AD._rows(pitched(hidden, pitch), torch.zeros(5, dtype=torch.int32))
    assert torch.equal(rows, hidden) and rows.stride(0) % 8 == 0 and ids.dtype == torch.int64
    assert (rows.stride(0) == pitch) == (pitch % 8 == 0)  # and no others


@pytest.mark.gpu
@pytest.mark.parametrize("pitch", [129, 130, 132, 136])
def test_any_pitch(pitch, cuda_device):
    *x, gen = make(40, 128, 700, 3, 16, "mixed", seed=1)
    labels = torch.randint(0, 700, (40,), generator=gen).to(cuda_device)
    h, w, a, b, s, ids = on(cuda_device, *x)
    assert torch.equal(AD.adapter_logits(pitched(h, pitch), w, a, b, s, ids), AD.adapter_logits(h, w, a, b, s, ids))
    grads = []
    for operand in (h.clone(), pitched(h, pitch)):
        lp, ent = AD.adapter_logprobs_from_hidden(operand.requires_grad_(), w, labels, a, b, s, ids)
        grads.append((lp.detach(), ent.detach()) + torch.autograd.grad(lp.sum() + ent.sum(), operand))
    assert all(torch.equal(p, q) for p, q in zip(*grads))
