"""Beam search (``skyrl_amd.beam_search``) against the definitions in 64 bits.

Parents and tokens are compared exactly.  That holds where totals of different beams differ by more than the operator's error -- 2^-23 relative to a
sum of exponentials, so 1.2e-7 in its logarithm, and the cast of a score -- which the cases with random logits have by their size (some thousand
gaps of 1e-3 and more) and the others by construction.  A score is one rounding of 2^-24 of a total, and that error: |total| 2^-24 + 2e-7.
"""

from __future__ import annotations

import math

import pytest
import torch

from skyrl_amd import beam_search as BS

pytestmark = pytest.mark.gpu
BF16, F32, INF, NAN = torch.bfloat16, torch.float32, math.inf, math.nan


def plain(logits, scores, k, temperature=1.0):
    z, s = logits.double().cpu(), scores.double().cpu()
    N, B, V = z.shape
    y = z / temperature
    total = s[:, :, None] + y - torch.logsumexp(y, 2, keepdim=True)
    ended = (s == -INF) | (z == -INF).all(2)
    total[ended] = -INF
    total[(~torch.isfinite(z) & (z != -INF)).any(2) | s.isnan() | (s == INF)] = NAN
    flat = total.flatten(1)
    nan = flat.isnan()
    order = torch.sort(torch.where(nan, -INF, flat), dim=1, descending=True, stable=True).indices
    order = order.gather(1, torch.sort(nan.gather(1, order).to(torch.int8), dim=1, stable=True).indices)[:, :k]
    return flat.gather(1, order), order // V, order % V


def check(got, logits, scores, k, temperature=1.0):
    want, parents, tokens = plain(logits, scores, k, temperature)
    assert got.scores.dtype == F32 and got.parents.dtype == got.tokens.dtype == torch.int64
    assert torch.equal(got.parents.cpu(), parents) and torch.equal(got.tokens.cpu(), tokens)
    have = got.scores.double().cpu()
    odd = ~torch.isfinite(want)
    assert torch.equal(have[odd].nan_to_num(7.0, neginf=-9.0), want[odd].nan_to_num(7.0, neginf=-9.0))
    assert bool(((have - want)[~odd].abs() <= want[~odd].abs() * 2.0 ** -24 + 2e-7).all())


def some_logits(N, B, V, dtype, seed, device):
    gen = torch.Generator(device=device).manual_seed(seed)
    z = torch.randn(N, B, V, generator=gen, device=device) * 2.5
    at = torch.randint(0, V, (N, B, 6), generator=gen, device=device)
    z.scatter_add_(2, at, torch.rand(N, B, 6, generator=gen, device=device) * 12)
    return z.to(dtype), torch.rand(N, B, generator=gen, device=device) * -9


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,B,V,k", [(1, 1, 1, 1), (1, 1, 2, 2), (2, 3, 5, 15), (3, 4, 7, 9), (1, 4, 1000, 8), (2, 1, 4099, 128), (5, 7, 33001, 13), (1, 2, 151936, 4),
                                     (2, 8, 100003, 16), (1, 16, 70001, 64), (70, 8, 999, 16), (1, 128, 500, 128), (2, 100, 65537, 100), (300, 2, 20000, 4)])
def test_selection(cuda_device, N, B, V, k, dtype):
    logits, scores = some_logits(N, B, V, dtype, N + V, cuda_device)
    check(BS.beam_select(logits, scores, k), logits, scores, k)


@pytest.mark.parametrize("temperature", [0.3, 0.7, 1.7, 1e-4, 1e4])
def test_temperature(cuda_device, temperature):
    logits, scores = some_logits(3, 5, 52001, F32, 1, cuda_device)
    check(BS.beam_select(logits, scores, 10, temperature=temperature), logits, scores, 10, temperature)


@pytest.mark.parametrize("V,k", [(600, 40), (60001, 20), (17, 17)])
def test_equal_totals_go_to_the_lower_beam_and_token(cuda_device, V, k):
    for logits in (torch.zeros(2, 4, V), torch.randint(0, 2, (2, 1, V)).float().expand(2, 4, V), torch.randint(0, 3, (2, 4, 1)).float().expand(2, 4, V)):
        logits = logits.to(cuda_device)
        scores = torch.tensor([[-1.0, -1.0, -0.5, -0.5], [-2.0, -2.0, -2.0, -2.0]], device=cuda_device)
        check(BS.beam_select(logits, scores, k), logits, scores, k)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [9, 700, 70001])
def test_masks_and_ended_beams(cuda_device, V, dtype):
    """Rows with few logits, one or none; scores of -inf; all of an item's beams ended."""
    logits, scores = some_logits(4, 6, V, dtype, V, cuda_device)
    logits[0, 0, :] = -INF
    logits[0, 1, 1:] = -INF
    logits[0, 2, : V - 2] = -INF
    logits[1, :, 3:] = -INF
    scores[0, 3] = scores[1, 0] = -INF
    scores[2] = -INF
    logits[3] = -INF
    for k in (1, 3, 9):
        check(BS.beam_select(logits, scores, k), logits, scores, k)


@pytest.mark.parametrize("V", [11, 70001])
def test_nan_and_infinities_sort_behind(cuda_device, V):
    logits, scores = some_logits(4, 5, V, F32, V, cuda_device)
    logits[0, 1, V // 2] = NAN
    logits[1, 0, 0] = INF
    scores[2, 3], scores[2, 4] = NAN, INF
    logits[3, :, V - 1] = NAN
    logits[3, 2, 0] = INF
    scores[3, 1] = -INF
    for k in (1, 4, 12, 30):
        check(BS.beam_select(logits, scores, k), logits, scores, k)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_masks_of_the_lowest_value_and_far_logits(cuda_device, dtype):
    V = 70001
    logits, scores = some_logits(3, 4, V, F32, 5, cuda_device)
    logits = logits.to(dtype)
    lowest = torch.finfo(dtype).min
    logits[0, :, 100:] = lowest
    logits[0, 1, :] = lowest           # all of a row: uniform
    logits[1, 0] += 30000.0
    logits[1, 1, 5:] = -1e10
    logits[2, 2] = -3e38
    logits[2, 2, 77] = 3e38
    check(BS.beam_select(logits, scores, 12), logits, scores, 12)


def test_the_order_of_totals_that_differ_in_the_last_bits(cuda_device):
    """Beams of the same logits and scores 2e-6 apart, 2 units of the last place of what comes back: in the order of their scores all the same."""
    V = 50000
    logits = torch.randn(1, 1, V, device=cuda_device).expand(1, 8, V)
    scores = (-12.0 - torch.tensor([3.0, 1, 7, 0, 2, 6, 5, 4], device=cuda_device) * 2e-6)[None]
    got = BS.beam_select(logits, scores, 8)
    assert got.parents.tolist() == [[3, 1, 4, 0, 7, 6, 5, 2]]
    check(got, logits, scores, 8)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_of_any_pitch(cuda_device, dtype):
    big, _ = some_logits(6, 9, 5003, dtype, 2, cuda_device)
    scores = torch.rand(6, 9, device=cuda_device)
    for logits, s in ((big[::2, 1:8:3, 1:4000], scores[::2, 1:8:3]), (big.transpose(0, 1)[:, :4, 3:], scores.t()[:, :4]), (big[:, :, ::2], scores),
                      (big[:1].expand(4, 9, 5003), scores[:4])):
        check(BS.beam_select(logits, s, 6), logits, s, 6)


def test_a_row_beyond_32_bit_offsets(cuda_device):
    big = torch.zeros(3, 2, 1 << 30, dtype=BF16, device=cuda_device)[:, :, 5:60005]
    logits, scores = some_logits(3, 2, 60000, BF16, 9, cuda_device)
    big.copy_(logits)
    check(BS.beam_select(big, scores, 5), logits, scores, 5)


def test_no_prompts(cuda_device):
    got = BS.beam_select(torch.empty(0, 3, 10, device=cuda_device), torch.empty(0, 3, device=cuda_device), 2)
    assert all(t.shape == (0, 2) for t in got)


def test_selection_replays_from_a_graph_and_runs_on_another_stream(cuda_device):
    logits, scores = some_logits(4, 4, 80001, BF16, 0, cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        BS.beam_select(logits, scores, 8)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    state = torch.arange(16.0, device=cuda_device)[:, None].expand(16, 33).contiguous()
    with torch.cuda.graph(graph):
        got = BS.beam_select(logits, scores, 4)
        moved = BS.beam_reorder([state], got.parents)[0]
    for seed in range(1, 4):
        new, s = some_logits(4, 4, 80001, BF16, seed, cuda_device)
        logits.copy_(new), scores.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        eager = BS.beam_select(logits, scores, 4)
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        assert torch.equal(moved[:, 5].cpu(), (eager.parents + torch.arange(0, 16, 4, device=cuda_device)[:, None]).reshape(-1).float().cpu())
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            other = BS.beam_select(logits, scores, 4)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(other, eager))


# ------------------------------------------------------------------------------------------------------------- states


def moved(t, parents, B_in):
    N, B_out = parents.shape
    p = parents.cpu()
    has = (p >= 0) & (p < B_in)
    rows = (torch.where(has, p, 0) + torch.arange(N)[:, None] * B_in).reshape(-1)
    out = t.cpu()[rows]
    out[~has.reshape(-1)] = 0
    return out


def caches(rows, device, gen):
    """States as models have them, and odd ones: caches with room, both halves of one tensor, other types, odd sizes, transposed."""
    r = lambda *s, dtype=BF16: torch.randn(*s, generator=gen, device=device).to(dtype)  # noqa: E731
    both = r(rows, 2, 3, 20, 16)
    return [r(rows, 2, 40, 64)[:, :, :33], r(rows, 5, 7, dtype=F32), both[:, 0], both[:, 1], r(rows, 4, 12, 8)[:, 1:3, 2:9, :5], r(rows),
            torch.randint(0, 99, (rows, 3), device=device), torch.randint(0, 99, (rows, 17), device=device).to(torch.uint8), r(rows, 6, 9, 10).transpose(1, 3),
            r(9, rows, 8).transpose(0, 1), r(rows, 1, 2048)]


@pytest.mark.parametrize("N,B_in,B_out", [(1, 1, 1), (1, 4, 4), (3, 5, 2), (2, 1, 6), (7, 8, 8), (1, 130, 200)])
def test_states_follow_their_parents(cuda_device, N, B_in, B_out):
    gen = torch.Generator(device=cuda_device).manual_seed(N + B_in)
    states = caches(N * B_in, cuda_device, gen)
    parents = torch.randint(0, B_in, (N, B_out), generator=gen, device=cuda_device)
    for out in (None, [torch.empty_strided((N * B_out,) + t.shape[1:], t.stride(), dtype=t.dtype, device=cuda_device) if t.stride(0) >= t.stride(-1) and i not in (9,)
                       else torch.empty((N * B_out,) + t.shape[1:], dtype=t.dtype, device=cuda_device) for i, t in enumerate(states)]):
        got = BS.beam_reorder(states, parents, out=out)
        for t, u in zip(states, got):
            assert torch.equal(u.cpu(), moved(t, parents, B_in))


@pytest.mark.parametrize("N,B", [(1, 1), (1, 4), (6, 5), (2, 33), (1, 128)])
def test_states_in_place(cuda_device, N, B):
    gen = torch.Generator(device=cuda_device).manual_seed(B)
    for parents in (torch.randint(0, B, (N, B), generator=gen, device=cuda_device), torch.arange(B, device=cuda_device).expand(N, B),
                    torch.arange(B, device=cuda_device).flip(0).expand(N, B), torch.zeros(N, B, dtype=torch.int64, device=cuda_device),
                    torch.randint(-1, B + 1, (N, B), generator=gen, device=cuda_device)):
        states = caches(N * B, cuda_device, gen)
        want = [moved(t, parents, B) for t in states]
        got = BS.beam_reorder(states, parents, out=states)
        for t, u, w in zip(states, got, want):
            assert u is t and torch.equal(u.cpu(), w)


def test_parents_outside_give_zeros(cuda_device):
    t = torch.ones(6, 40, device=cuda_device)
    parents = torch.tensor([[0, -1, 2], [3, 1, 2 ** 62]], device=cuda_device)
    assert BS.beam_reorder([t], parents)[0][:, 0].tolist() == [1, 0, 1, 0, 1, 0]


def test_what_lies_beside_a_state_is_left(cuda_device):
    room = torch.arange(8 * 2 * 50 * 16, device=cuda_device, dtype=F32).reshape(8, 2, 50, 16)
    before = room.clone()
    parents = torch.tensor([[1, 0, 3, 3], [0, 0, 1, 2]], device=cuda_device)
    BS.beam_reorder([room[:, :, :31]], parents, out=[room[:, :, :31]])
    assert torch.equal(room[:, :, 31:], before[:, :, 31:])
    assert torch.equal(room[:, :, :31].cpu(), moved(before[:, :, :31], parents, 4))
    into = before.clone()
    BS.beam_reorder([before[:, :, 4:9]], parents, out=[into[:, :, 4:9]])
    assert torch.equal(into[:, :, :4], before[:, :, :4]) and torch.equal(into[:, :, 9:], before[:, :, 9:])


def test_more_states_than_one_launch_holds(cuda_device):
    states = [torch.full((4, 3), float(i), device=cuda_device) + torch.arange(4, device=cuda_device)[:, None] for i in range(450)]
    got = BS.beam_reorder(states, torch.tensor([[3, 3], [0, 1]], device=cuda_device).reshape(1, 4))
    assert all(t[:, 2].tolist() == [i + 3.0, i + 3.0, i + 0.0, i + 1.0] for i, t in enumerate(got))


def test_states_beyond_32_bit_offsets(cuda_device):
    t = torch.zeros(3, 1 << 31, dtype=torch.uint8, device=cuda_device)
    t[:, -5:] = torch.tensor([1, 2, 3], device=cuda_device, dtype=torch.uint8)[:, None]
    parents = torch.tensor([[2, 0, 0]], device=cuda_device)
    assert BS.beam_reorder([t], parents)[0][:, -3].tolist() == [3, 1, 1]
    BS.beam_reorder([t], parents, out=[t])
    assert t[:, -1].tolist() == [3, 1, 1]


def test_the_op_under_the_dispatcher(cuda_device):
    logits, scores = some_logits(2, 3, 40, F32, 3, cuda_device)
    torch.library.opcheck(BS.logits_beam_select, (logits, scores, 4, 1.0), test_utils=("test_schema", "test_faketensor"))


def test_autograd_sees_what_is_written(cuda_device):
    """A state that an eager graph has saved and that is then reordered in place: its backward refuses."""
    t = torch.randn(4, 3, device=cuda_device)
    w = torch.randn(4, 3, device=cuda_device, requires_grad=True)
    loss = (w * t).sum()
    before = t._version
    BS.beam_reorder([t], torch.tensor([[1, 0, 2, 3]], device=cuda_device), out=[t])
    assert t._version > before
    with pytest.raises(RuntimeError):
        loss.backward()


def test_results_that_share_memory_with_states_are_refused(cuda_device):
    base = torch.arange(40.0, device=cuda_device).reshape(10, 4)
    parents = torch.zeros(1, 4, dtype=torch.int64, device=cuda_device)
    for states, out in (([base[:4]], [base[2:6]]), ([base[:4], base[4:8]], [base[4:8], base[:4]]), ([base[:4], base[:4].clone()], [torch.empty_like(base[:4])] * 2),
                        ([base[:4], base[:4]], [base[:4], base[:4]]), ([base[:4], base[4:8]], [base[:4], base[1:5]])):
        with pytest.raises(ValueError):
            BS.beam_reorder(states, parents, out=out)
    wide = torch.zeros(130, 2, device=cuda_device)
    with pytest.raises(ValueError):  # in place at most 128 beams
        BS.beam_reorder([wide], torch.zeros(1, 130, dtype=torch.int64, device=cuda_device), out=[wide])
    got = BS.beam_reorder([base[:4]], parents, out=[base[6:]])  # beside each other in one tensor
    assert torch.equal(got[0], base[:1].expand(4, 4))
