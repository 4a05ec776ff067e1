"""How many runs of memory the rows of a state are taken as.  No GPU."""

from __future__ import annotations

import itertools
import random

import pytest
import torch

from skyrl_amd import beam_search as BS


def launches(state, out):
    return BS._layout(state.shape, state.stride(), out.stride(), state.dtype, 2, state.shape[0] // 2).launches


def bf16(*shape):
    return torch.empty(shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("state,segments,nbytes", [
    (bf16(4, 500, 4, 128).transpose(1, 2), 1, 500 * 4 * 128 * 2),          # [rows, length, heads, dim] seen as [rows, heads, length, dim]
    (bf16(4, 512, 4, 128)[:, :500].transpose(1, 2), 1, 500 * 4 * 128 * 2),
    (bf16(4, 2, 512, 64)[:, :, :137], 2, 137 * 64 * 2),
    (bf16(4, 3, 70, 40).transpose(2, 3), 1, 3 * 70 * 40 * 2),               # the innermost dimension is not the last
    (bf16(4, 5, 6, 7, 8).permute(0, 3, 1, 4, 2), 1, 5 * 6 * 7 * 8 * 2),
    (bf16(4, 9, 10)[:, :, ::2], 45, 2),
])
def test_a_row_is_as_few_runs_as_its_memory_is(state, segments, nbytes):
    ((sizes, places),) = launches(state, state)
    assert sizes[4:] == (segments, nbytes) and places == ((0, 0),)


def test_the_longest_dimension_is_the_one_that_is_stepped_through():
    """From [rows, length, heads, dim] into [rows, heads, length, dim]: 4 places of 500 segments, not 500 of 4."""
    ((sizes, places),) = launches(bf16(4, 500, 4, 128).transpose(1, 2), bf16(4, 4, 500, 128))
    assert sizes[4:] == (500, 256) and len(places) == 4


def test_every_element_is_taken_to_its_place():
    """Random shapes, orders, gaps and results, walked as the kernel walks them."""
    rng = random.Random(3)
    for _ in range(400):
        dims = rng.randint(1, 4)
        shape = [rng.choice([1, 2, 3, 5]) for _ in range(dims)]

        def view():
            order, room = rng.sample(range(dims), dims), [n + rng.choice([0, 0, 1, 2]) for n in shape]
            t = torch.zeros([1 + rng.randint(0, 1)] + [room[i] for i in order], dtype=torch.int32)
            t = t.permute(0, *[1 + order.index(i) for i in range(dims)])
            return t[(slice(None),) + tuple(slice(n) for n in shape)]

        state, out = view()[:1], view()[:1]
        if rng.random() < 0.2 and shape[0] > 1:
            state = state[:, :1].expand(1, *shape)
        places = set()
        found = list(BS._layout(state.shape, state.stride(), out.stride(), state.dtype, 1, 1).launches)
        for (_, step, _, to_step, n, nbytes), starts in found:
            for (at, to_at), i, byte in itertools.product(starts, range(n), range(0, nbytes, 4)):
                places.add((at + i * step + byte, to_at + i * to_step + byte))
        index = itertools.product(*(range(n) for n in shape))
        want = {(4 * sum(i * s for i, s in zip(x, state.stride()[1:])), 4 * sum(i * s for i, s in zip(x, out.stride()[1:]))) for x in index}
        assert places == want
