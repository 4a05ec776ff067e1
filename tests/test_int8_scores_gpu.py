"""Log-probabilities of the head in 8-bit integers (``skyrl_amd.int8_head``) where the integer sums and the places of rows are at their limits, against the
definition in 64 bits: bounds that a wrong sum, a wrong row or a missing one would exceed by far."""

from __future__ import annotations

import math

import pytest
import torch

from skyrl_amd import int8_head as I

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def check(lp, ent, y, labels, unit):
    logp = torch.log_softmax(y, 1)
    want, entropy = logp.gather(1, labels[:, None])[:, 0], -(logp.exp() * logp).sum(1)
    assert bool(((lp.double().cpu() - want).abs() <= unit).all()), (lp.double().cpu() - want).abs().max()
    assert bool(((ent.double().cpu() - entropy).abs() <= 10 * unit).all()), (ent.double().cpu() - entropy).abs().max()


@pytest.mark.parametrize("T", [1, 16, 40, 64, 130, 300])
def test_scores_of_the_largest_sums(cuda_device, T):
    """Weights of -128 and 127 at the largest hidden size, scaled by 2^-20: logits of -16 to 16 from sums of up to 127 * 128 * H.  A logit is off by 2^-22 of
    itself (the sum's rounding, two products and a scale of 2^-24 each), the label's and the others'; exponentials and their sum by 1e-5."""
    H, V = I.MAX_HIDDEN, 70
    values = torch.full((V, H), -128, dtype=torch.int8, device=cuda_device)
    cut = [128 * ((v * 13) % V) * (H // 128) // V for v in range(V)]
    for v in range(V):
        values[v, :cut[v]] = 127
    head = I.Int8Head(values, torch.full((V,), 2.0 ** -20, device=cuda_device))
    hidden = torch.ones(T, H, device=cuda_device)
    hidden[T // 2:] = -1
    sums = torch.tensor([127.0 * c - 128.0 * (H - c) for c in cut], dtype=torch.float64) * 127
    assert 127 * 128 * H == -sums.min() < 2 ** 31
    y = torch.sign(hidden[:, :1].double().cpu()) * sums * 2.0 ** -20 / 127
    labels = torch.arange(T) * 7 % V
    lp, ent = I.int8_logprobs_from_hidden(hidden, head, labels.to(cuda_device))
    check(lp, ent, y, labels, 2.0 ** -22 * 2 * float(y.abs().max()) + 1e-5)


@pytest.mark.parametrize("T", [5, 500])
def test_scores_beyond_32_bit_offsets(cuda_device, T):
    """4.8 GB of values, four of them not zero: each label's row and all statistics in closed form.  Sums are of some 600 fp32 additions one after the other (36719
    partials in 64 streams, or 4.7 M rows in 256 workgroups of 8 waves and 4 rows a lane), and of few behind that: off by 700 2^-24 = 4e-5 and the exponentials'
    1e-5; labels' logits are 2 apart."""
    V, H = 4_700_000, 1024
    values = torch.zeros(V, H, dtype=torch.int8, device=cuda_device)
    at = torch.tensor([0, V // 2, 4_194_304, V - 1], device=cuda_device)
    values[at, 0] = torch.tensor([4, 5, 6, 7], dtype=torch.int8, device=cuda_device)
    head = I.Int8Head(values, torch.full((V,), 2.0 ** -6, device=cuda_device))
    hidden = torch.zeros(T, H, device=cuda_device, dtype=BF16)
    hidden[:, 0] = 127.0 * (1 + torch.arange(T, device=cuda_device) % 2)  # logits of 8 to 14, or 16 to 28
    labels = torch.cat([at, torch.tensor([1], device=cuda_device)])[torch.arange(T, device=cuda_device) // 2 % 5]
    lp, ent = I.int8_logprobs_from_hidden(hidden, head, labels)
    z = torch.tensor([4.0, 5, 6, 7], dtype=torch.float64)[None] * hidden[:, :1].double().cpu() * 2.0 ** -6
    lse = torch.log(torch.exp(z).sum(1) + (V - 4))
    picked = torch.cat([z, torch.zeros(T, 1, dtype=torch.float64)], 1)[torch.arange(T), torch.arange(T) // 2 % 5]
    entropy = lse - (torch.exp(z - lse[:, None]) * z).sum(1)
    assert bool(((lp.double().cpu() - (picked - lse)).abs() <= 1e-4).all()), (lp.double().cpu() - (picked - lse)).abs().max()
    assert bool(((ent.double().cpu() - entropy).abs() <= 1e-3).all()), (ent.double().cpu() - entropy).abs().max()
    assert math.isclose(float(lse[0]), math.log(sum(math.exp(127 * i / 64) for i in (4, 5, 6, 7)) + V - 4))
