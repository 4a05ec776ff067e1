"""Rows of finite logits far from zero in ``top_logprobs_from_logits``: a mask of the type's lowest value or of -1e10, in a whole row or in all of it that
one wave sees, and large offsets.  Only a row without any logit above -inf is empty.

Order is compared exactly.  Tolerances: a log-probability is a difference of logits times 1 / temperature, each with a rounding of 2^-24, and the logarithm
of a sum of at most V terms: 4 roundings relative to the value, 2^-22, and 5e-5 as for other rows; a value beyond fp32 is infinite.  The
entropy as for other rows, 1e-4.  Gradients: as for other rows, eps / 2 + 2e-5 of the value and 2e-5 of the coefficients times p, 2e-6 of
the coefficients where a column has a term of its own; up to |lse| = 4096 the fp32 lse costs p up to 2^-11 of its value (two roundings of 2^-24 * 4096 each,
in base 2), which the sizes here stay away from.

The 64-bit definitions are taken of z minus the row's largest z, which changes none of the results and which 64 bits hold exactly for values of one
size: of z itself they lose the logarithm of a sum from 2^53 on (the step at 1e20 is 16384).
"""

from __future__ import annotations

import math

import pytest
import torch

from skyrl_amd import torch_utils as TU
from test_top_logits_gpu import INF, plain, plain_grad

pytestmark = pytest.mark.gpu
LOWEST = "lowest"


def rows(kind, value, T, V, dtype, gen):
    """Ordinary logits of which some or all are `value`; labels are ordinary where a row has any such."""
    low = torch.finfo(dtype).min if value == LOWEST else value
    logits = torch.randn(T, V, generator=gen) * 2.5
    labels = torch.randint(0, V, (T,), generator=gen)
    if kind == "whole":
        logits[:] = low
    elif kind == "two levels":  # the higher one has all of the probability
        logits = torch.where(torch.rand(T, V, generator=gen) < 0.5, low, low * 0.75)
    elif kind == "all but one":
        keep = logits.gather(1, labels[:, None])
        logits[:] = low
        logits.scatter_(1, labels[:, None], keep)
    elif kind == "most":
        gone = torch.rand(T, V, generator=gen) < 0.995
        gone.scatter_(1, labels[:, None], False)
        logits[gone] = low
    elif kind == "mixed with -inf":
        logits[:] = low
        logits[:, ::3] = -INF
    return logits.to(dtype), labels


def shifted(logits):
    z = logits.double()
    top = z.amax(1, keepdim=True)
    return z - torch.where(torch.isfinite(top), top, 0.0)


def near(got, want, tol):
    """Where fp32 holds the value; an infinity where it does not."""
    got, want = got.detach().cpu().double(), want.double()
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, want.sign() * INF, want)
    same = got == want
    assert bool((same | ((got - want).abs() <= tol + want.abs() * 2.0**-22)).all()), (got - want)[~same][:4]


@pytest.mark.parametrize("kind", ["whole", "two levels", "all but one", "most", "mixed with -inf"])
@pytest.mark.parametrize("value", [-1e4, -1e9, -1e10, -1e20, -1e30, LOWEST])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks_of_finite_values(kind, value, dtype, cuda_device):
    gen = torch.Generator().manual_seed(3)
    for V in (300, 33001, 66001):  # singles and few pieces; a workgroup for a row; workgroups that share one, and their join
        logits, labels = rows(kind, value, 5, V, dtype, gen)
        labels[1] = -100
        for temperature in (1.0, 0.3, 2.0):
            got = TU.top_logprobs_from_logits(logits.to(cuda_device), labels.to(cuda_device), 20, temperature=temperature)
            want = plain(shifted(logits), labels, 20, temperature)
            assert torch.equal(got.top_ids.cpu(), want["top_ids"]) and torch.equal(got.ranks.cpu(), want["ranks"])
            near(got.logprobs, want["logprobs"], 5e-5)
            near(got.top_logprobs, want["top_logprobs"], 5e-5)
            near(got.entropy, want["entropy"], 1e-4)


@pytest.mark.parametrize("offset", [-1e30, -1e10, -1e6, 1e6, 1e10, 1e30, 3.3e38])
@pytest.mark.parametrize("V", [4099, 70001])
def test_large_offsets(offset, V, cuda_device):
    """A few steps of the type apart, at either end of its range."""
    gen = torch.Generator().manual_seed(5)
    base = torch.tensor(offset)
    step = (torch.nextafter(base.abs(), torch.tensor(INF)) - base.abs()) * base.sign()
    logits = base - step.abs() * torch.randint(0, 3, (4, V), generator=gen)
    labels = torch.randint(0, V, (4,), generator=gen)
    for temperature in (1.0, 0.3):
        got = TU.top_logprobs_from_logits(logits.to(cuda_device), labels.to(cuda_device), 5, temperature=temperature)
        want = plain(shifted(logits), labels, 5, temperature)
        assert torch.equal(got.top_ids.cpu(), want["top_ids"]) and torch.equal(got.ranks.cpu(), want["ranks"])
        near(got.logprobs, want["logprobs"], 5e-5)
        near(got.top_logprobs, want["top_logprobs"], 5e-5)
        near(got.entropy, want["entropy"], 1e-4)


@pytest.mark.parametrize("value", [-1e6, -1e9, -1e10, -1e30, LOWEST])
@pytest.mark.parametrize("kind", ["whole", "two levels", "most", "mixed with -inf"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", ["g", "q", "h", "gqh"])
def test_gradients_of_such_rows(value, kind, dtype, which, cuda_device):
    gen = torch.Generator().manual_seed(7)
    for T, V, k in ((4, 700, 5), (3, 20011, 20)):
        logits, labels = rows(kind, value, T, V, dtype, gen)
        labels[0] = -1
        g = torch.randn(T, generator=gen) if "g" in which else None
        q = torch.randn(T, generator=gen) * 0.1 if "q" in which else None
        h = torch.randn(T, k, generator=gen) if "h" in which else None
        for temperature in (1.0, 0.3):
            d, y = logits.to(cuda_device), labels.to(cuda_device)
            at = lambda t: None if t is None else t.to(cuda_device)  # noqa: E731
            lp, ent, lse, pz, ranks, top, ids = TU.logits_top_fwd(d, y, k, 1.0 / temperature)
            assert bool(torch.isfinite(lse).all()) and bool(torch.isfinite(pz).all())
            got = TU.logits_top_bwd(d, y, lse, pz, at(g), at(q), ids, at(h), 1.0 / temperature).cpu().double()
            want = plain_grad(shifted(logits), labels, k, temperature, g, q, h)
            w = plain(shifted(logits), labels, k, temperature)
            coefficient = sum(t.double().abs().reshape(T, -1).sum(1) for t in (g, h) if t is not None) + torch.zeros(T)
            coefficient = ((coefficient + (0 if q is None else 40 * q.double().abs())) / temperature)[:, None]
            own = torch.zeros_like(want).scatter_(1, w["top_ids"], 1.0)
            own[torch.arange(T), labels.clamp(0)] = 1.0
            bound = want.abs() * (torch.finfo(dtype).eps / 2 + 2e-5) + 2e-5 * coefficient * w["p"] + 2e-6 * coefficient * own + 1e-30
            assert bool(((got - want).abs() <= bound).all()), ((got - want).abs() - bound).max()


def test_rows_that_are_not_numbers_stay_that_way(cuda_device):
    """+inf and NaN beside far logits: no finite answer is made up; an empty row stays empty."""
    for V in (1000, 66001):
        z = torch.full((5, V), torch.finfo(torch.float32).min)
        z[0, 3], z[1, 3], z[2, 3] = INF, math.nan, -INF
        z[3], z[4] = -INF, -INF
        z[4, 9] = math.nan
        y = torch.full((5,), 7)
        r = TU.top_logprobs_from_logits(z.to(cuda_device), y.to(cuda_device), 2)
        lp, ent = r.logprobs.cpu(), r.entropy.cpu()
        assert bool(torch.isnan(ent[[0, 1, 4]]).all()) and not bool(torch.isfinite(lp[[0, 1, 4]]).any())
        assert abs(float(lp[2]) + math.log(V - 1)) < 5e-5 and abs(float(ent[2]) - math.log(V - 1)) < 1e-4
        assert float(lp[3]) == -INF and float(ent[3]) == 0.0 and r.top_ids[3].tolist() == [0, 1] and r.top_ids[0, 0] == 3
