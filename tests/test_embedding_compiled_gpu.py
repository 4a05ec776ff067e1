"""``embedding_lookup`` and the other operators around the head inside a compiled program: one graph without a break, the same results and gradients."""

from __future__ import annotations

import pytest
import torch

from skyrl_amd import beam_search as BS
from skyrl_amd import embedding as E
from skyrl_amd import int8_head as I

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_lookup_in_a_compiled_step(cuda_device, dtype, backend):
    weight = torch.randn(300, 72, device=cuda_device, dtype=dtype).requires_grad_()
    ids = torch.randint(-1, 301, (5, 9), device=cuda_device)
    mix = torch.randn(72, 72, device=cuda_device, dtype=dtype)

    def step(w, i):
        return torch.tanh(E.embedding_lookup(w, i, scale=0.5, padding_idx=3) @ mix)

    compiled = torch.compile(step, backend=backend, fullgraph=True, dynamic=False)
    d = torch.randn(5, 9, 72, device=cuda_device, dtype=dtype)
    for _ in range(2):
        want, got = step(weight, ids), compiled(weight, ids)
        assert torch.equal(want, got)
        (a,), (b,) = torch.autograd.grad(want, weight, d), torch.autograd.grad(got, weight, d)
        assert torch.equal(a, b)
        ids = torch.randint(-1, 301, (5, 9), device=cuda_device)


def test_a_decoding_step_in_a_compiled_program(cuda_device):
    """Lookup, 8-bit logits and the selection; the states are reordered outside, as they have to be."""
    table = torch.randn(500, 128, device=cuda_device, dtype=torch.bfloat16)
    head = I.quantize_head(table)

    def step(ids, scores):
        h = E.embedding_lookup(table, ids)
        z = I.int8_logits(h, head)
        best = BS.beam_select(z.reshape(2, 3, 500), scores, 4)
        return best.scores, best.parents, best.tokens

    with torch.no_grad():
        compiled = torch.compile(step, backend="aot_eager", fullgraph=True, dynamic=False)
        ids, scores = torch.randint(0, 500, (6,), device=cuda_device), torch.randn(2, 3, device=cuda_device)
        assert all(torch.equal(a, b) for a, b in zip(step(ids, scores), compiled(ids, scores)))


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_what_works_on_addresses_leaves_a_compiled_program(cuda_device, backend):
    """``beam_reorder`` and ``embedding_backward_accumulate`` between two compiled parts of a program."""
    parents = torch.tensor([[1, 0, 3, 3]], device=cuda_device)
    d, ids = torch.randn(3, 8, device=cuda_device), torch.tensor([0, 2, 2], device=cuda_device)

    def step(cache, buffer):
        doubled = cache * 2
        new = BS.beam_reorder([doubled], parents)[0]
        BS.beam_reorder([cache], parents, out=[cache])
        E.embedding_backward_accumulate(d * 2, ids, buffer)
        return new + 1, cache - 1, buffer * 3

    def inputs():
        return torch.arange(12.0, device=cuda_device).reshape(4, 3), torch.ones(5, 8, device=cuda_device)

    compiled = torch.compile(step, backend=backend, dynamic=False)
    with torch.no_grad():
        for _ in range(2):
            assert all(torch.equal(a, b) for a, b in zip(step(*inputs()), compiled(*inputs())))
