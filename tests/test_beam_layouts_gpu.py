"""States whose dimensions lie in memory in another order than their shape's: results, and that they take about as long as plain indexing does."""

from __future__ import annotations

import pytest
import torch

from skyrl_amd import beam_search as BS
from test_beam_segments_gpu import least_ms, moved, values

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16

LAYOUTS = {
    "length before heads": ((512, 4, 128), lambda t: t[:, :500].transpose(1, 2)),
    "dim before length": ((4, 500, 128), lambda t: t.transpose(2, 3)),
    "length last, with room": ((4, 128, 512), lambda t: t[:, :, :, :501]),
    "all turned round": ((64, 50, 4, 16), lambda t: t.permute(0, 4, 2, 3, 1)),
}


@pytest.mark.parametrize("layout", sorted(LAYOUTS))
def test_states_in_any_order_of_dimensions(cuda_device, layout):
    shape, view = LAYOUTS[layout]
    parents = torch.tensor([[1, 0, 2, 2], [3, -1, 0, 1]], device=cuda_device)
    t = view(values((8, *shape), BF16, cuda_device, 1))
    want = moved(t, parents, 4)
    (new,) = BS.beam_reorder([t], parents)
    assert torch.equal(new, want) and new.is_contiguous()
    for like in (t, want.contiguous()):  # into the same strides, and into those of the shape's order
        out = torch.empty_strided(like.shape, like.stride(), dtype=BF16, device=cuda_device)
        BS.beam_reorder([t], parents, out=[out])
        assert torch.equal(out, want)
    BS.beam_reorder([t], parents, out=[t])
    assert torch.equal(t, want)


@pytest.mark.parametrize("layout", sorted(LAYOUTS))
def test_they_take_about_as_long_as_plain_indexing_at_most(cuda_device, layout):
    shape, view = LAYOUTS[layout]
    states = [view(values((128, *shape), BF16, cuda_device, i)) for i in range(8)]
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    parents = torch.randint(0, 8, (16, 8), generator=gen, device=cuda_device)
    rows = (parents + torch.arange(0, 128, 8, device=cuda_device)[:, None]).reshape(-1)
    into = [torch.empty_strided(t.shape, t.stride(), dtype=BF16, device=cuda_device) for t in states]
    own, inside = least_ms(lambda: BS.beam_reorder(states, parents, out=into)), least_ms(lambda: BS.beam_reorder(states, parents, out=states))
    plain = least_ms(lambda: [t[rows] for t in states])
    assert own <= 1.5 * plain and inside <= 1.5 * plain, (own, inside, plain)  # both at the memory's rate; element by element it was 8 to 1000 times as long
