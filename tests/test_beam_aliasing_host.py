"""Which results of a reordering are refused because they share memory with what is read or written beside them.  No GPU: everything is refused in front
of the look at the device, and what is not refused ends there (RuntimeError)."""

from __future__ import annotations

import random

import pytest
import torch

from skyrl_amd import beam_search as BS

P = torch.tensor([[1, 2, 3, 0]])


def cases():
    buf = torch.zeros(16, 40)
    kv = torch.zeros(4, 2, 3, 20, 16)                       # keys and values side by side
    late = torch.zeros(4, 20, 2, 3, 16)                     # the same in each position
    flat = torch.zeros(4, 100)                              # several states of a row in one run
    both = torch.zeros(4, 2, 12, 8)
    ids = torch.zeros(4, 8, dtype=torch.int64)
    a, b, c, p = buf[:4], buf[4:8], buf[8:12], ids[0, :4].view(1, 4)
    return {
        "in place, read for another result too": ([a, a], [a, b], P, True),
        "the same, of another layout": ([a, a.view(4, 8, 5)], [a, torch.zeros(4, 8, 5)], P, True),
        "in place twice": ([a, a], [a, a], P, True),
        "in place, columns of another state in place": ([a, a[:, 2:]], [a, a[:, 2:]], P, True),
        "results that overlap each other": ([c, buf[12:]], [buf[:4], buf[2:6]], P, True),
        "results that interleave and share columns": ([a[:, :10], b[:, :10]], [c[:, :10], c[:, 9:19]], P, True),
        "a result on another state": ([a, b], [b, c], P, True),
        "a result beside its state": ([buf[:4]], [buf[2:6]], P, True),
        "a result on its state in other strides": ([torch.zeros(4, 4)], [torch.zeros(4, 4)], P, False),
        "the transposed state": ([flat[:, :4]], [flat[:, :4].t()], P, True),
        "a result on the parents": ([torch.zeros(4, 1, dtype=torch.int64)], [ids[:1, :4].t()], p, True),
        "parents inside a state in place": ([ids], [ids], p, True),
        "beside each other": ([a, b], [a, b], P, False),
        "into other rows": ([a, b], [c, buf[12:]], P, False),
        "the same state twice": ([a, a], [b, c], P, False),
        "both halves in place": ([kv[:, 0], kv[:, 1]], [kv[:, 0], kv[:, 1]], P, False),
        "both halves of each position in place": ([late[:, :, 0], late[:, :, 1]], [late[:, :, 0], late[:, :, 1]], P, False),
        "the used part of both": ([kv[:, 0, :, :7], kv[:, 1, :, :7]], [kv[:, 0, :, :7], kv[:, 1, :, :7]], P, False),
        "one half in place, the other into new memory": ([kv[:, 0], kv[:, 1]], [kv[:, 0], torch.zeros_like(kv[:, 1])], P, False),
        "one half into the other": ([kv[:, 0]], [kv[:, 1]], P, False),
        "heads apart, positions interleaved": ([late[:, :, :, :2], late[:, :, :, 2:]], [late[:, :, :, :2], late[:, :, :, 2:]], P, False),
        "states of a row of other shapes": ([flat[:, :24].view(4, 2, 3, 4), flat[:, 24:31], flat[:, 40:100].view(4, 3, 20)[:, :, 3:9]],
                                            [flat[:, :24].view(4, 2, 3, 4), flat[:, 24:31], flat[:, 40:100].view(4, 3, 20)[:, :, 3:9]], P, False),
        "transposed halves": ([both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)], [both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)], P, False),
        "parents beside a state in one tensor": ([ids[:, 4:]], [ids[:, 4:]], p, False),
        "an expanded state": ([torch.zeros(1, 5).expand(4, 5)], [a[:, :5]], P, False),
    }


@pytest.mark.parametrize("name", sorted(cases()))
def test_what_is_refused(name):
    states, out, parents, refused = cases()[name]
    with pytest.raises(ValueError if refused else RuntimeError) as e:
        BS.beam_reorder(states, parents, out=out)
    assert ("shares memory" in str(e.value)) == refused


def test_no_overlap_is_missed():
    """Random views of 60 elements against the elements that they have."""
    rng = random.Random(5)
    base = torch.arange(60, dtype=torch.int32)
    clashes = apart = 0
    for _ in range(4000):
        regions, held = [], []
        for _ in range(rng.choice([2, 2, 3, 4])):
            dims = rng.choice([1, 2, 2, 3])
            shape = tuple(rng.choice([1, 2, 3, 4]) for _ in range(dims))
            steps = tuple(rng.choice([0, 1, 2, 3, 4, 6, 8, 12]) for _ in range(dims))
            at = rng.randrange(12)
            if at + sum(s * (n - 1) for n, s in zip(shape, steps)) >= 60:
                continue
            reach = BS._reach(shape, steps, 4)
            is_result = rng.random() < 0.6
            regions.append((1000 + at * 4, 1000 + at * 4 + reach.extent, reach, is_result))
            held.append((set(base.as_strided(shape, steps, at).reshape(-1).tolist()), is_result))
        truly = any((x[1] or y[1]) and x[0] & y[0] for i, x in enumerate(held) for y in held[:i])
        said = BS._clash(regions)
        assert said or not truly, regions
        clashes, apart = clashes + truly, apart + (not said)
    assert clashes > 500 and apart > 500
