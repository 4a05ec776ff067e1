"""Which roundings the gradients of the head with adapters have: dz once to bf16, but for the label's value, and each result once.  u = s A h, du = s B^T dz
and what they are contracted with keep fp32's precision.

Bounds.  A result is round(true + e), e what the rounding of dz makes of it.  Both parts are known without the operator: r is the rounding of the true
result, d that of a dz rounded to bf16, brought through the products in 64 bits.  They are independent of each other, so the error's norm is
sqrt(r^2 + d^2) of the result's, give or take 1 / sqrt(2 n) of it for n values that carry the norm: n is 9600 at least here (dB, whose norm lies in the
label's rows: T R values), so that 5 % is seven times that.  An u or du of one bf16 term adds its own rounding, some 1.65e-3 of the norm where the
result's is 1.65e-3: more than a third, which the test on the CPU shows for each place that holds two terms.
"""

from __future__ import annotations

import pytest
import torch

from skyrl_amd import adapters as AD
from test_adapters_gpu import on

T, H, R, N = 300, 256, 32, 3
MARGIN = 1.05
PLACES = ("u in dB", "du in dA", "du in d_hidden")


def problem(V, entropy_grad):
    gen = torch.Generator().manual_seed(V)
    b16 = torch.bfloat16
    hidden = torch.randn(T, H, generator=gen).to(b16)
    weight = (torch.randn(V, H, generator=gen) * 0.002).to(b16)      # p is flat, and d_hidden is the adapters' part for the most
    a = (torch.randn(N, R, H, generator=gen) / 16).to(b16)
    b = (torch.randn(N, V, R, generator=gen) * 0.02).to(b16)
    scaling = 0.5 + torch.rand(N, generator=gen)
    ids = torch.randint(0, N, (T,), generator=gen)
    labels = torch.randint(0, V, (T,), generator=gen)
    g = torch.randn(T, generator=gen)
    q = 0.1 * torch.randn(T, generator=gen) if entropy_grad else None
    return (hidden, weight, a, b, scaling, ids), labels, g, q


def rounded(x):
    return x.to(torch.bfloat16).double()


def gradients(x, labels, g, q, round_dz, one_term=None):
    """By the formulas in 64 bits; the fourth is the weight's part of d_hidden.  round_dz: dz in bf16 but for the label's value; one_term: the place where a factor is one bf16 number."""
    h, w, a, b, s = (t.double() for t in x[:5])
    a, b, s = a[x[5]], b[x[5]], s[x[5]]  # of each token
    u = s[:, None] * torch.einsum("trh,th->tr", a, h)
    z = h @ w.T + torch.einsum("tvr,tr->tv", b, u)
    lsm = torch.log_softmax(z, 1)
    p = lsm.exp()
    dz = -p * g.double()[:, None]
    if q is not None:
        dz -= q.double()[:, None] * p * (lsm - (p * lsm).sum(1, keepdim=True))
    rows = torch.arange(T)
    dz[rows, labels] += g.double()
    if round_dz:
        exact = dz[rows, labels]
        dz = rounded(dz)
        dz[rows, labels] = exact
    du = s[:, None] * torch.einsum("tvr,tv->tr", b, dz)
    at = lambda place, t: rounded(t) if one_term == place else t  # noqa: E731
    per_token = torch.nn.functional.one_hot(x[5], N).double()
    product = dz @ w
    d_hidden = product + torch.einsum("trh,tr->th", a, at("du in d_hidden", du))
    d_a = torch.einsum("tn,tr,th->nrh", per_token, at("du in dA", du), h)
    d_b = torch.stack([(dz * per_token[:, n:n + 1]).T @ at("u in dB", u) for n in range(N)])
    return d_hidden, d_a, d_b, product


def errors(got, want):
    return [float((g.double() - w).norm() / w.norm()) for g, w in zip(got, want[:3])]


def bounds(case):
    want = gradients(*case, round_dz=False)
    r = errors([rounded(t) for t in want], want)
    d = errors(gradients(*case, round_dz=True), want)
    return want, [MARGIN * (x * x + y * y) ** 0.5 for x, y in zip(r, d)]


CASES = [(V, e) for V in (300, 2049) for e in (False, True)]  # d_hidden of a transposed weight, and of one that is read in place


@pytest.mark.parametrize("V,entropy_grad", CASES)
def test_the_bounds_hold_two_roundings_and_not_a_third(V, entropy_grad):
    case = problem(V, entropy_grad)
    want, bound = bounds(case)
    assert all(e <= b for e, b in zip(errors([rounded(t) for t in gradients(*case, round_dz=True)], want), bound))
    for place, k in zip(PLACES, (2, 1, 0)):
        off = errors([rounded(t) for t in gradients(*case, round_dz=True, one_term=place)], want)
        assert off[k] > 1.1 * bound[k], (place, off[k], bound[k])


@pytest.mark.gpu
@pytest.mark.parametrize("V,entropy_grad", CASES)
def test_gradients_are_rounded_once(V, entropy_grad, cuda_device):
    x, labels, g, q = case = problem(V, entropy_grad)
    want, bound = bounds(case)
    if V < 1024:  # d_hidden of a transposed weight is rounded before the adapters' part joins it, and twice that way
        more = float((rounded(want[3]) - want[3]).norm() / want[0].norm())
        bound[0] = (bound[0] ** 2 + (MARGIN * more) ** 2) ** 0.5
    d, y = on(cuda_device, *x), labels.to(cuda_device)
    _, _, lse, pz = AD.lmhead_adapter_fwd(d[0], d[1], y, *d[2:], 1.0)
    got = AD.lmhead_adapter_bwd(d[0], d[1], y, *d[2:], lse, pz, g.to(cuda_device), None if q is None else q.to(cuda_device), 1.0)
    for name, off, most in zip(("d_hidden", "d_lora_a", "d_lora_b"), errors([t.cpu() for t in got], want), bound):
        print(name, off, most)
        assert off <= most, (name, off, most)
