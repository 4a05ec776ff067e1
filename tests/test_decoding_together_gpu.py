"""The embedding, the head in 8-bit integers and beam search as a decoder uses them together, and a tied table in training.

The "model" is one recurrent layer, s' = (s + E[token]) / 2, on 32-bit states, with a head quantised from the embedding's table."""

from __future__ import annotations

import math

import pytest
import torch

from skyrl_amd import beam_search as BS
from skyrl_amd import embedding as E
from skyrl_amd import int8_head as I
from skyrl_amd import torch_utils as TU
from skyrl_amd.fused_linear_logprob_hip import linear_cross_entropy

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
N, B, V, H, STEPS = 3, 4, 20011, 200, 7


def model(device):
    gen = torch.Generator().manual_seed(11)
    table = (torch.randn(V, H, generator=gen) * 0.5).to(BF16).to(device)
    return table, I.quantize_head(table), torch.randn(N, H, generator=gen).to(device)


def step(table, head, state, cache, scores, tokens):
    """One step of all beams: new state, cache, scores, tokens and parents."""
    state = (state + E.embedding_lookup(table, tokens).float()) / 2
    logits = I.int8_logits(state, head, dtype=F32)
    picked = BS.beam_select(logits.reshape(N, -1, V), scores, B)
    state, cache = BS.beam_reorder([state, cache], picked.parents)
    return state, cache, picked, logits


def test_beams_of_a_small_model(cuda_device):
    """Every selection is that of the logits in 64 bits; the scores that come out are those of the sequences, scored anew."""
    table, head, start = model(cuda_device)
    state, tokens = start, torch.arange(5, 5 + N, device=cuda_device)
    scores = torch.zeros(N, 1, device=cuda_device)
    cache = torch.zeros(N, 2, STEPS, 3, device=cuda_device, dtype=BF16)
    history = tokens[:, None]
    for i in range(STEPS):
        before = cache.clone()
        state, cache, picked, logits = step(table, head, state, cache, scores, tokens)
        beams = scores.shape[1]
        total = scores.double()[:, :, None] + torch.log_softmax(logits.double().reshape(N, beams, V), 2)
        best, at = total.flatten(1).sort(dim=1, descending=True, stable=True)
        assert torch.equal(picked.parents, at[:, :B] // V) and torch.equal(picked.tokens, at[:, :B] % V)
        assert float((picked.scores - best[:, :B]).abs().max()) < 1e-5
        rows = (picked.parents + torch.arange(N, device=cuda_device)[:, None] * beams).reshape(-1)
        assert torch.equal(cache, before[rows])
        scores, tokens = picked.scores, picked.tokens.reshape(-1)
        cache[:, :, i] = (tokens % 256).to(BF16)[:, None, None]  # what a real cache would keep of the token
        history = torch.cat([history[rows], tokens[:, None]], 1)
    assert torch.equal(cache[:, 0, :, 0], (history[:, 1:] % 256).to(BF16))  # the cache went the way of its beam
    # The sequences once more, all positions at once.
    rows = E.embedding_lookup(table, history[:, :-1]).float()
    s, hidden = start.repeat_interleave(B, 0), []
    for i in range(STEPS):
        s = (s + rows[:, i]) / 2
        hidden.append(s)
    logprobs, entropy = I.int8_logprobs_from_hidden(torch.stack(hidden, 1), head, history[:, 1:])
    assert float((logprobs.double().sum(1) - scores.reshape(-1).double()).abs().max()) < 1e-4
    last = TU.top_logprobs_from_logits(logits, torch.zeros(N * B, dtype=torch.int64, device=cuda_device), 1)
    parents = (picked.parents + torch.arange(N, device=cuda_device)[:, None] * B).reshape(-1)
    assert float((last.entropy[parents] - entropy[:, -1]).abs().max()) < 1e-4


def test_a_step_replays_from_a_graph(cuda_device):
    table, head, start = model(cuda_device)
    state, tokens = start.repeat_interleave(B, 0), torch.arange(N * B, device=cuda_device)
    scores, cache = torch.zeros(N, B, device=cuda_device), torch.randn(N * B, 2, 9, 8, device=cuda_device).to(BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(table, head, state, cache, scores, tokens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(table, head, state, cache, scores, tokens)
    for seed in range(4):
        gen = torch.Generator(device=cuda_device).manual_seed(seed)
        tokens.copy_(torch.randint(0, V, tokens.shape, generator=gen, device=cuda_device))
        scores.copy_(torch.randn(scores.shape, generator=gen, device=cuda_device))
        cache.copy_(torch.randn(cache.shape, generator=gen, device=cuda_device))
        graph.replay()
        torch.cuda.synchronize()
        want = step(table, head, state, cache, scores, tokens)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[3], want[3])
        assert all(torch.equal(a, b) for a, b in zip(got[2], want[2]))


def test_two_steps_at_once_on_two_streams(cuda_device):
    table, head, start = model(cuda_device)
    args = [(start + i, torch.randn(N, 2, 9, 8, device=cuda_device), torch.zeros(N, 1, device=cuda_device), torch.arange(N, device=cuda_device) + i) for i in range(2)]
    want = [step(table, head, *a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(step(table, head, *a))
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) and all(torch.equal(a, b) for a, b in zip(x[2], y[2]))


def test_a_tied_table_in_training(cuda_device):
    """Loss of a head whose weight is the embedding's table: the leaf's gradient has both parts.  Tolerance: two gradients in bf16, each rounded once, their sum
    rounded once more: 3 * 2^-9 of the parts' magnitudes, and the head's own 2e-3 of the largest (its gradient takes dz and hidden states in bf16)."""
    T, H2, V2 = 90, 128, 700
    gen = torch.Generator().manual_seed(2)
    table = (torch.randn(V2, H2, generator=gen) * 0.3).to(BF16).to(cuda_device).requires_grad_()
    ids, labels = (torch.randint(0, V2, (T,), generator=gen).to(cuda_device) for _ in range(2))
    hidden = E.embedding_lookup(table, ids, scale=2.0)
    logprobs, _ = linear_cross_entropy(hidden, table, labels, 1.0)
    (-logprobs.mean()).backward()

    t = table.detach().double().requires_grad_()
    h = t[ids] * 2
    h16 = h + (h.to(BF16).double() - h).detach()
    loss = -torch.log_softmax(h16 @ t.T, 1).gather(1, labels[:, None]).mean()
    loss.backward()
    off = (table.grad.double() - t.grad).abs()
    assert float(off.max()) <= 2e-3 * float(t.grad.abs().max()) + 3 * 2.0 ** -9 * float(t.grad.abs().max())
    assert math.isfinite(float(off.max())) and float(torch.nn.functional.cosine_similarity(table.grad.double().flatten(), t.grad.flatten(), dim=0)) > 0.9999
