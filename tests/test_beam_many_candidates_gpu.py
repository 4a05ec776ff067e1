"""Selections of many candidates, as many as 128, from few and many sorted lists: results, and that they take no longer than elementary operations do."""

from __future__ import annotations

import math

import pytest
import torch

from skyrl_amd import beam_search as BS
from test_beam_search_gpu import check, some_logits

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


# One list, fewer lists than candidates, about as many, and more; lists shorter than k.
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,B,V,k", [(1, 1, 9000, 128), (1, 1, 151936, 127), (1, 3, 40007, 100), (2, 4, 151936, 128), (1, 8, 151936, 128), (3, 16, 70001, 128), (1, 128, 5, 128),
                                     (1, 100, 40, 128), (2, 65, 16411, 65), (2, 2, 130, 128), (600, 1, 300, 128)])
def test_many_candidates(cuda_device, N, B, V, k, dtype):
    logits, scores = some_logits(N, B, V, dtype, V + k, cuda_device)
    check(BS.beam_select(logits, scores, k), logits, scores, k)
    if B > 1:  # ended beams, and one so far behind that only its head is near
        scores[0, B - 1] = -math.inf
        scores[-1, 0] -= 6.0
        check(BS.beam_select(logits, scores, k), logits, scores, k)


@pytest.mark.parametrize("V", [700, 40009, 151936])
def test_many_equal_candidates(cuda_device, V):
    """All of a row's logits equal, or two values in turns: the lower columns of the lower beams."""
    for logits in (torch.zeros(2, 5, V), (torch.arange(V) % 2).float().expand(2, 5, V), (torch.arange(V) >= V // 2).float().expand(2, 5, V)):
        logits = logits.to(cuda_device)
        scores = torch.tensor([[-1.0, -1.0, -3.0, -1.0, -math.inf], [0.0, -0.5, 0.0, -0.5, 0.0]], device=cuda_device)
        check(BS.beam_select(logits, scores, 128), logits, scores, 128)


def test_candidates_that_all_come_from_one_list(cuda_device):
    """The best of a row in one part of it, those of another beam spread evenly."""
    V = 151936
    logits = torch.randn(1, 4, V, device=cuda_device)
    logits[0, 2, 80000:80200] += 30.0 + torch.rand(200, device=cuda_device)
    scores = torch.tensor([[-2.0, -2.5, -2.25, -9.0]], device=cuda_device)
    check(BS.beam_select(logits, scores, 128), logits, scores, 128)


def elementary(logits, scores, k):
    y = logits.double()
    total = (scores.double()[:, :, None] + torch.log_softmax(y, 2)).flatten(1)
    best, at = total.sort(dim=1, descending=True, stable=True)
    return best[:, :k], at[:, :k]


def least_ms(f):
    f()
    times = []
    for _ in range(7):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(5):
            f()
        end.record()
        end.synchronize()
        times.append(begin.elapsed_time(end) / 5)
    return min(times)


@pytest.mark.parametrize("B,ended", [(1, False), (4, False), (4, True), (8, True)])
def test_many_candidates_take_no_longer_than_elementary_operations(cuda_device, B, ended):
    logits, scores = some_logits(1, B, 151936, BF16, B, cuda_device)
    if ended:
        scores[0, B - 1] = -math.inf
    own, plain = least_ms(lambda: BS.beam_select(logits, scores, 128)), least_ms(lambda: elementary(logits, scores, 128))
    assert own <= plain, (own, plain)
