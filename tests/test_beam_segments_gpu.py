"""States whose rows are segments of any length at any alignment: results, what lies beside them, and that they take no longer than elementary operations do."""

from __future__ import annotations

import pytest
import torch

from skyrl_amd import beam_search as BS

pytestmark = pytest.mark.gpu
BF16, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


def values(shape, dtype, device, seed):
    gen = torch.Generator(device=device).manual_seed(seed)
    return torch.randint(0, 251, shape, generator=gen, device=device).to(dtype)


def moved(t, parents, B_in):
    N = parents.shape[0]
    has = ((parents >= 0) & (parents < B_in)).reshape(-1)
    rows = (torch.where(has.view(parents.shape), parents, 0) + torch.arange(0, N * B_in, B_in, device=t.device)[:, None]).reshape(-1)
    out = t[rows]
    out[~has] = 0
    return out


@pytest.mark.parametrize("dtype", [U8, BF16, F32])
@pytest.mark.parametrize("begin", [0, 1, 3, 8])
@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 64, 81, 257])
def test_segments_of_any_length_and_place(cuda_device, width, begin, dtype):
    room = values((12, 5, width + 11), dtype, cuda_device, width)
    for parents in (torch.tensor([[1, 0, 2, 2], [3, 3, 0, 1], [0, 1, 2, 3]], device=cuda_device), torch.tensor([[-1, 0, 4, 2]] * 3, device=cuda_device)):
        for cut in (slice(None), slice(1, 4)):
            t = room[:, cut, begin:begin + width]
            want = moved(t, parents, 4)
            assert torch.equal(BS.beam_reorder([t], parents)[0], want)
            into = values(room.shape, dtype, cuda_device, 77)
            after = into.clone()
            after[:, cut, begin:begin + width] = want
            BS.beam_reorder([t], parents, out=[into[:, cut, begin:begin + width]])
            assert torch.equal(into, after)
            if begin + width + 2 <= room.shape[2]:  # into another alignment
                wide = values((12, 5, width + 13), dtype, cuda_device, 78)
                after = wide.clone()
                after[:, cut, 2:2 + width] = want
                BS.beam_reorder([t], parents, out=[wide[:, cut, 2:2 + width]])
                assert torch.equal(wide, after)
            inside = room.clone()
            after = room.clone()
            after[:, cut, begin:begin + width] = want
            BS.beam_reorder([inside[:, cut, begin:begin + width]], parents, out=[inside[:, cut, begin:begin + width]])
            assert torch.equal(inside, after)


@pytest.mark.parametrize("dtype,shape,cut", [(BF16, (8, 3, 700, 81), 501), (U8, (8, 3, 900, 33), 601), (BF16, (8, 40, 130, 64), 3), (F32, (8, 2, 64, 1300), 1299)])
def test_many_segments_and_long_ones(cuda_device, dtype, shape, cut):
    room = values(shape, dtype, cuda_device, cut)
    parents = torch.tensor([[1, 0, 1, 1], [2, 3, 0, 2]], device=cuda_device)
    for t in (room[:, :, :cut], room[:, :, 1:, : shape[3] - 1]):
        want = moved(t, parents, 4)
        assert torch.equal(BS.beam_reorder([t], parents)[0], want)
        inside = room.clone()
        after = room.clone()
        view = inside.as_strided(t.shape, t.stride(), t.storage_offset())
        after.as_strided(t.shape, t.stride(), t.storage_offset()).copy_(want)
        BS.beam_reorder([view], parents, out=[view])
        assert torch.equal(inside, after)


def least_ms(f):
    f()
    times = []
    for _ in range(7):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(3):
            f()
        end.record()
        end.synchronize()
        times.append(begin.elapsed_time(end) / 3)
    return min(times)


@pytest.mark.parametrize("shape,cut", [((128, 4, 512, 81), (slice(None), slice(501), slice(None))), ((128, 4, 128, 512), (slice(None), slice(None), slice(17))),
                                       ((128, 4, 128, 512), (slice(None), slice(None), slice(501))), ((128, 64, 512, 8), (slice(None), slice(500), slice(4)))])
def test_short_and_odd_segments_take_no_longer_than_elementary_operations(cuda_device, shape, cut):
    states = [values(shape, BF16, cuda_device, i)[(slice(None), *cut)] for i in range(8)]
    into = [torch.empty(shape, dtype=BF16, device=cuda_device)[(slice(None), *cut)] for _ in range(8)]
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    parents = torch.randint(0, 8, (16, 8), generator=gen, device=cuda_device)
    rows = (parents + torch.arange(0, 128, 8, device=cuda_device)[:, None]).reshape(-1)

    def plain():
        for t, u in zip(states, into):
            u.copy_(t[rows])

    own = least_ms(lambda: BS.beam_reorder(states, parents, out=into))
    assert own <= least_ms(plain), own
