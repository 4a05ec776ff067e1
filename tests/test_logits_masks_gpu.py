"""Masks of finite values in the statistics of materialised logits (``logprobs_and_entropy_from_logits``): where a thread has seen nothing else, its sum
has to vanish beside the row's ordinary logits.

Tolerances as for other rows: four roundings of 2^-24 relative to at most 40 and the sum of at most V / 512 + 20 terms a thread, below 5e-5;
the entropy's products reach 60, 1e-4.  Gradients: p has the error of its exponent, 2^-24 * 64, the result one rounding: eps / 2 + 2e-5 of the
value, 2e-5 of the coefficient times p, and 2e-6 of the coefficient at the label, where two terms may cancel.
"""

from __future__ import annotations

import math

import pytest
import torch

from skyrl_amd import torch_utils as TU

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [-1e9, -1e10, -1e15, -1e20, -1e30, "lowest", -math.inf])
@pytest.mark.parametrize("share", [0.5, 0.97, 1.0])  # 1.0: all but the label
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_rows(value, share, dtype, cuda_device):
    gen = torch.Generator().manual_seed(2)
    for T, V in ((4, 1), (5, 3001), (3, 33001)):
        z = torch.randn(T, V, generator=gen) * 2.5
        labels = torch.randint(0, V, (T,), generator=gen)
        gone = torch.rand(T, V, generator=gen) < share
        gone.scatter_(1, labels[:, None], False)
        z[gone] = torch.finfo(dtype).min if value == "lowest" else value
        z = z.to(dtype)
        g, q = torch.randn(T, generator=gen), torch.randn(T, generator=gen) * 0.1
        for temperature in (1.0, 0.3):
            y = z.double() / temperature
            lsm = torch.log_softmax(y, 1)
            p = lsm.exp()
            logp = torch.where(p > 0, lsm, 0.0)
            want_lp, want_ent = lsm.gather(1, labels[:, None])[:, 0], -(p * logp).sum(1)
            d = z.to(cuda_device).requires_grad_()
            lp, ent = TU.logprobs_and_entropy_from_logits(d, labels.to(cuda_device), temperature=temperature)
            assert float((lp.detach().cpu().double() - want_lp).abs().max()) <= 5e-5
            assert float((ent.detach().cpu().double() - want_ent).abs().max()) <= 1e-4
            (got,) = torch.autograd.grad((lp, ent), d, (g.to(cuda_device), q.to(cuda_device)))
            want = -p * g.double()[:, None] - q.double()[:, None] * p * (logp + want_ent[:, None])
            want.scatter_add_(1, labels[:, None], g.double()[:, None])
            want /= temperature
            coefficient = ((g.double().abs() + 40 * q.double().abs()) / temperature)[:, None]
            own = torch.zeros_like(want).scatter_(1, labels[:, None], 1.0)
            bound = want.abs() * (torch.finfo(dtype).eps / 2 + 2e-5) + 2e-5 * coefficient * p + 2e-6 * coefficient * own + 1e-30
            assert bool(((got.cpu().double() - want).abs() <= bound).all())


def test_not_a_number_is_not_lost(cuda_device):
    """A thread whose logits are NaN and masked ones beside threads with larger logits."""
    z = torch.full((2, 40001), -1e10)
    z[:, 17] = 3.0
    z[1, 39999] = math.nan
    for x in (z, z.to(torch.bfloat16)):
        lp, ent = TU.logprobs_and_entropy_from_logits(x.to(cuda_device), torch.tensor([17, 17], device=cuda_device))
        assert abs(float(lp[0])) <= 5e-5 and bool(torch.isnan(lp[1])) and bool(torch.isnan(ent[1]))
