"""States of so many short segments that one grid does not hold them (2^32 threads): rows, beams of one item and segments of one row go in several launches."""

from __future__ import annotations

import pytest
import torch

from skyrl_amd import beam_search as BS

pytestmark = pytest.mark.gpu


def state(rows, segments, device):
    """One byte of every two."""
    gen = torch.Generator(device=device).manual_seed(rows)
    return torch.randint(0, 256, (rows, segments, 2), generator=gen, device=device, dtype=torch.uint8)


def moved(t, parents, B_in):
    N = parents.shape[0]
    return t[(parents + torch.arange(0, N * B_in, B_in, device=t.device)[:, None]).reshape(-1)]


# rows by several launches of items; one item's beams by several; one row's segments by several
@pytest.mark.parametrize("N,B_in,B_out,segments", [(171, 3, 3, 32801), (1, 3, 515, 32801), (5, 2, 150, 40009), (1, 2, 2, (1 << 24) + 77)])
def test_into_other_rows(cuda_device, N, B_in, B_out, segments):
    assert N * B_out * segments >= 1 << 24
    t = state(N * B_in, segments, cuda_device)
    parents = torch.randint(0, B_in, (N, B_out), device=cuda_device)
    (got,) = BS.beam_reorder([t[:, :, 0]], parents)
    assert torch.equal(got, moved(t, parents, B_in)[:, :, 0])
    del got
    if N * B_out < 300:
        out = state(N * B_out, segments, cuda_device)
        beside = out[:, :, 0].clone()
        BS.beam_reorder([t[:, :, 0]], parents, out=[out[:, :, 1]])
        assert torch.equal(out[:, :, 1], moved(t, parents, B_in)[:, :, 0]) and torch.equal(out[:, :, 0], beside)


@pytest.mark.parametrize("N,B,segments", [(515, 2, 32801), (1, 2, (1 << 24) + 77)])
def test_in_place(cuda_device, N, B, segments):
    t = state(N * B, segments, cuda_device)
    parents = torch.randint(0, B, (N, B), device=cuda_device)
    parents[-1] = torch.tensor([1, 0], device=cuda_device)
    beside, want = t[:, :, 0].clone(), moved(t, parents, B)[:, :, 1]
    BS.beam_reorder([t[:, :, 1]], parents, out=[t[:, :, 1]])
    assert torch.equal(t[:, :, 1], want) and torch.equal(t[:, :, 0], beside)
