"""Labels outside the vocabulary in the head with adapters: the log-probability is the constant 0, and so its gradient is 0.

Expected values differentiate what the operator returns, in 64 bits on the same bf16 operands.  Tolerances, norm by norm of a token's d_hidden and an
adapter's dA and dB: dz is rounded to bf16 once (2^-8 at most, half a step), each result once, and p has the logits' error twice over.
"""

from __future__ import annotations

import math

import pytest
import torch

from skyrl_amd import adapters as AD
from test_adapters_gpu import E, TRAIN, make, on, plain_logits, row_norms, z_error

pytestmark = pytest.mark.gpu

OUTSIDE = (-100, -1, 2**40, -(2**63))


def outside(labels, V, gen, share=0.3):
    """Labels of which some lie outside: padding of several kinds, and the first column behind the vocabulary."""
    kinds = torch.tensor(OUTSIDE + (V,))
    return torch.where(torch.rand(labels.shape, generator=gen) < share, kinds[torch.randint(0, len(kinds), labels.shape, generator=gen)], labels)


@pytest.mark.parametrize("T,H,V,N,R,order,temperature", TRAIN)
@pytest.mark.parametrize("entropy_grad", [False, True])
def test_the_gradient_is_that_of_the_returned_value(T, H, V, N, R, order, temperature, entropy_grad, cuda_device):
    *x, gen = make(T, H, V, N, R, order, seed=T + V + R)
    labels = outside(torch.randint(0, V, (T,), generator=gen), V, gen)
    labels[0] = -100
    has = (labels >= 0) & (labels < V)
    g, q = torch.randn(T, generator=gen), torch.randn(T, generator=gen) * 0.1
    leaves = [x[i].double().requires_grad_() for i in (0, 2, 3)]
    z = plain_logits(leaves[0], x[1], leaves[1], leaves[2], x[4], x[5]) / temperature
    lsm = torch.log_softmax(z, 1)
    want_lp = torch.where(has, lsm.gather(1, labels.clamp(0, V - 1)[:, None])[:, 0], 0.0)
    want_ent = -(lsm.exp() * lsm).sum(1)
    loss = (want_lp * g).sum() + ((want_ent * q).sum() if entropy_grad else 0.0)
    want = torch.autograd.grad(loss, leaves)

    d = on(cuda_device, *x)
    dl = [d[i].clone().requires_grad_() for i in (0, 2, 3)]
    lp, ent = AD.adapter_logprobs_from_hidden(dl[0], d[1], labels.to(cuda_device), dl[1], dl[2], d[4], d[5], temperature=temperature)
    z_err = float(z_error(*x).max()) / temperature
    assert float((lp.detach().cpu().double() - want_lp.detach()).abs().max()) <= 2 * z_err + 5e-5
    assert not bool(lp.detach().cpu()[~has].any())
    assert float((ent.detach().cpu().double() - want_ent.detach()).abs().max()) <= 4 * z_err * (1 + math.log(V)) + 5e-5
    back = (lp * g.to(cuda_device)).sum() + ((ent * q.to(cuda_device)).sum() if entropy_grad else 0.0)
    got = torch.autograd.grad(back, dl)
    for mine, true in zip(got, want):
        row_norms(mine, true, 2 * E + 2 * z_err, 1e-6 * float(true.norm()) + 1e-12)
    if not entropy_grad:
        assert not bool(got[0][~has.to(cuda_device)].any())


@pytest.mark.parametrize("T,V", [(9, 300), (40, 2049), (300, 1111), (33000, 260)])  # d_hidden both ways; more tokens than one block
@pytest.mark.parametrize("entropy_grad", [False, True])
def test_such_tokens_are_tokens_without_a_gradient_on_the_logprob(T, V, entropy_grad, cuda_device):
    """The same bits as with that gradient zero, whatever it is: NaN too."""
    *x, gen = make(T, 64, V, 3, 8, "mixed", seed=T)
    labels = outside(torch.randint(0, V, (T,), generator=gen), V, gen)
    labels[-1] = V
    has = (labels >= 0) & (labels < V)
    g = torch.randn(T, generator=gen)
    q = torch.randn(T, generator=gen).mul(0.1).to(cuda_device) if entropy_grad else None
    d, y = on(cuda_device, *x), labels.to(cuda_device)
    _, _, lse, pz = AD.lmhead_adapter_fwd(d[0], d[1], y, *d[2:], 1.0)
    want = AD.lmhead_adapter_bwd(d[0], d[1], y, *d[2:], lse, pz, torch.where(has, g, 0.0).to(cuda_device), q, 1.0)
    for other in (g, torch.where(has, g, math.nan), torch.where(has, g, math.inf)):
        got = AD.lmhead_adapter_bwd(d[0], d[1], y, *d[2:], lse, pz, other.to(cuda_device), q, 1.0)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    if not entropy_grad:
        none = AD.lmhead_adapter_bwd(d[0], d[1], torch.full_like(y, -100), *d[2:], lse, pz, g.to(cuda_device), None, 1.0)
        assert not any(bool(t.any()) for t in none)
