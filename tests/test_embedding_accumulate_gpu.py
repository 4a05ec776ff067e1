"""Accumulation of the table's gradient into an fp32 buffer: windows of ids that are all different, rows of any size, and what it costs."""

from __future__ import annotations

import pytest
import torch

from skyrl_amd import embedding as E
from test_embedding_gpu import check_gradient
from test_lookup_node_gpu import least_us

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,H,V", [(1, 1, 3), (16, 3, 40), (16, 9, 16), (17, 64, 33), (40, 511, 64), (40, 513, 41), (31, 1030, 30), (500, 260, 16)])
def test_buffers_that_hold_something(cuda_device, T, H, V, dtype):
    """Each id once and runs of ids, several pieces and slices of a row with ends that repeat elements; twice into the same buffer."""
    gen = torch.Generator().manual_seed(T * H)
    d = torch.randn(T, H, generator=gen).to(dtype).to(cuda_device)
    for ids in (torch.randperm(max(T, V), generator=gen)[:T] % V, torch.arange(T) // 3 % V, torch.randint(-1, V + 1, (T,), generator=gen)):
        ids = ids.to(cuda_device)
        start = torch.randn(V, H, generator=gen).to(cuda_device)
        buffer = start.clone()
        E.embedding_backward_accumulate(d, ids, buffer, scale=0.5)
        check_gradient(buffer, d, ids, V, 0.5, start=start)
        once = buffer.clone()
        E.embedding_backward_accumulate(d, ids, buffer, scale=0.5)
        check_gradient(buffer, d, ids, V, 0.5, start=once)


def test_it_takes_no_longer_than_adding_row_by_row(cuda_device):
    ids = (151936 ** torch.rand(4096, device=cuda_device, dtype=torch.float64)).long().sub_(1).clamp_(0, 151935)
    d, buffer = torch.randn(4096, 2048, device=cuda_device, dtype=BF16), torch.zeros(151936, 2048, device=cuda_device)
    own, plain = least_us(lambda: E.embedding_backward_accumulate(d, ids, buffer)), least_us(lambda: buffer.index_add_(0, ids, d.float()))
    assert own <= plain, (own, plain)
