"""Embedding rows and the gradient of their table (``skyrl_amd.embedding``) against the definitions in 64 bits.

Tolerances.  A row is one fp32 product, rounded once: eps / 2 of the type and 2^-24.  A gradient element is a sum of n fp32 terms (n additions and
one product: (n + 1) 2^-24 of the sum of magnitudes) rounded once.
"""

from __future__ import annotations

import pytest
import torch

from skyrl_amd import embedding as E
from skyrl_amd import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def plain_rows(weight, ids, scale):
    w, ids = weight.double().cpu(), ids.cpu()
    has = (ids >= 0) & (ids < w.shape[0])
    return torch.where(has[..., None], w[torch.where(has, ids, 0)] * torch.tensor(scale, dtype=F32).double(), 0.0)


def plain_gradient(d_out, ids, vocab, scale, padding=None):
    """The gradient, the sums of magnitudes and the counts, 64 bits."""
    d, ids = d_out.double().cpu().reshape(-1, d_out.shape[-1]), ids.cpu().reshape(-1)
    takes = (ids >= 0) & (ids < vocab)
    if padding is not None:
        takes &= ids != padding % vocab
    s = torch.tensor(scale, dtype=F32).double()
    zeros = torch.zeros(vocab, d.shape[1], dtype=torch.float64)
    grad = zeros.clone().index_add_(0, ids[takes], d[takes]) * s
    size = zeros.clone().index_add_(0, ids[takes], d[takes].abs()) * s.abs()
    return grad, size, torch.bincount(ids[takes], minlength=vocab).double()[:, None]


def check_rows(out, weight, ids, scale):
    want = plain_rows(weight, ids, scale)
    bound = (torch.finfo(weight.dtype).eps / 2 + 2.0 ** -23) * want.abs() + torch.finfo(weight.dtype).smallest_normal
    assert out.dtype == weight.dtype and out.shape == want.shape
    assert bool(((out.double().cpu() - want).abs() <= bound).all())


def check_gradient(got, d_out, ids, vocab, scale, padding=None, start=None):
    want, size, n = plain_gradient(d_out, ids, vocab, scale, padding)
    bound = (n + 2) * 2.0 ** -24 * size + torch.finfo(got.dtype).eps / 2 * want.abs() * (1 + 1e-3) + torch.finfo(got.dtype).smallest_normal
    if start is not None:
        want = want + start.double().cpu()
        bound = bound + 2.0 ** -24 * want.abs()
    assert got.shape == want.shape
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), (float((off - bound).max()), (off > bound).nonzero()[:4].tolist())


def some_ids(kind, T, V, gen):
    if kind == "one":
        return torch.full((T,), V // 2, dtype=torch.int64)
    if kind == "apart":
        return torch.randperm(max(T, V), generator=gen)[:T] % V
    if kind == "text":
        return (V ** torch.rand(T, generator=gen, dtype=torch.float64)).long().sub_(1).clamp_(0, V - 1)
    if kind == "rising":
        return torch.arange(T) * V // max(1, T)
    if kind == "some outside":
        ids = torch.randint(-2, V + 2, (T,), generator=gen)
        ids[::7] = 2 ** 62
        ids[1::9] = -(2 ** 63)
        return ids
    if kind == "none":
        return torch.full((T,), -100, dtype=torch.int64)
    raise ValueError(kind)


SIZES = [(1, 1, 1), (1, 8, 5), (2, 3, 2), (15, 7, 40), (16, 64, 33), (17, 520, 9), (33, 9, 1000), (64, 257, 300), (65, 4, 70), (300, 1023, 257), (1000, 65, 33001),
         (611, 130, 1)]


@pytest.mark.parametrize("kind", ["one", "apart", "text", "rising", "some outside", "none"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,H,V", SIZES)
def test_rows_and_gradient(cuda_device, T, H, V, dtype, kind):
    gen = torch.Generator().manual_seed(T * 31 + H)
    weight = torch.randn(V, H, generator=gen).to(dtype).to(cuda_device).requires_grad_()
    ids = some_ids(kind, T, V, gen).to(cuda_device)
    d = torch.randn(T, H, generator=gen).to(dtype).to(cuda_device)
    out = E.embedding_lookup(weight, ids, scale=0.3)
    check_rows(out, weight.detach(), ids, 0.3)
    (grad,) = torch.autograd.grad(out, weight, d)
    assert grad.dtype == dtype
    check_gradient(grad, d, ids, V, 0.3)
    assert torch.equal(grad, E.lmhead_embedding_bwd(d, ids, V, 0.3, -1))


@pytest.mark.parametrize("kind", ["one", "apart", "text", "some outside"])
@pytest.mark.parametrize("T", [4095, 4096, 4097, 8192, 20001])
def test_more_tokens_than_a_sorted_block(cuda_device, T, kind):
    gen = torch.Generator().manual_seed(T)
    ids = some_ids(kind, T, 5003, gen).to(cuda_device)
    d = torch.randn(T, 72, generator=gen).to(BF16).to(cuda_device)
    check_gradient(E.lmhead_embedding_bwd(d, ids, 5003, 1.0, -1), d, ids, 5003, 1.0)


@pytest.mark.parametrize("order", ["rising", "falling", "interleaved"])
def test_sorting_keeps_the_order_of_equal_ids(cuda_device, order):
    """1 + 2^-24 + 2^-24 ... : the sum shows the order in which fp32 terms are added, so two runs and another place of the tokens agree."""
    T, V = 9000, 3
    ids = torch.arange(T) % V if order == "interleaved" else torch.arange(T) * V // T
    ids = (ids.flip(0) if order == "falling" else ids).to(cuda_device)
    d = torch.rand(T, 16, device=cuda_device) * 2.0 ** torch.randint(-20, 20, (T, 1), device=cuda_device)
    first = E.lmhead_embedding_bwd(d, ids, V, 1.0, -1)
    check_gradient(first, d, ids, V, 1.0)
    for _ in range(3):
        assert torch.equal(first, E.lmhead_embedding_bwd(d, ids, V, 1.0, -1))
    # the same tokens under ids that sort the same
    assert torch.equal(first, E.lmhead_embedding_bwd(d, ids * 11, 40, 1.0, -1)[[0, 11, 22]])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,H,V", [(1, 5, 3), (40, 64, 7), (300, 1023, 257), (5000, 36, 900)])
def test_accumulation_touches_the_named_rows_alone(cuda_device, T, H, V, dtype):
    gen = torch.Generator().manual_seed(T + H)
    ids = some_ids("text", T, V, gen)
    ids[T // 3:T // 2] = V  # outside
    ids = ids.to(cuda_device)
    d = torch.randn(T, H, generator=gen).to(dtype).to(cuda_device)
    start = torch.randn(V, H, generator=gen).to(cuda_device)
    named = torch.zeros(V, dtype=torch.bool, device=cuda_device)
    named[ids[(ids < V) & (ids != 0)]] = True
    start[~named] = float("nan")
    buffer = start.clone()
    out = E.embedding_backward_accumulate(d, ids, buffer, scale=2.0, padding_idx=0)
    assert out.data_ptr() == buffer.data_ptr()
    assert torch.equal(buffer[~named].isnan(), torch.ones_like(buffer[~named], dtype=torch.bool))
    keep = named.cpu()
    clean = torch.where(named[:, None], start, 0.0)
    check_gradient(torch.where(named[:, None], buffer, 0.0), d, ids, V, 2.0, padding=0, start=clean)
    assert int(keep.sum()) > 0 or T == 1


def test_a_tied_table_takes_both_gradients(cuda_device):
    """The head's dW and the embedding's in one fp32 buffer, as a trainer with tied weights accumulates them."""
    T, H, V = 70, 128, 500
    gen = torch.Generator().manual_seed(5)
    w = torch.randn(V, H, generator=gen).to(BF16).to(cuda_device)
    ids, labels = torch.randint(0, V, (T,), generator=gen).to(cuda_device), torch.randint(0, V, (T,), generator=gen).to(cuda_device)
    hidden, d = torch.randn(T, H, generator=gen).to(BF16).to(cuda_device), torch.randn(T, H, generator=gen).to(BF16).to(cuda_device)
    g = torch.randn(T, generator=gen).to(cuda_device)
    _, _, lse, _ = ops.lmhead_fwd(hidden, w, labels, 1.0, False)
    buffer = torch.zeros(V, H, device=cuda_device)
    ops.lmhead_bwd_accumulate(hidden, w, labels, lse, None, g, None, 1.0, buffer)
    head = buffer.clone()
    E.embedding_backward_accumulate(d.reshape(7, 10, H), ids.reshape(7, 10), buffer)
    check_gradient(buffer, d, ids, V, 1.0, start=head)


@pytest.mark.parametrize("padding", [0, 3, 299, -1])
def test_the_padding_row_takes_no_gradient(cuda_device, padding):
    ids = torch.randint(0, 300, (5, 41), device=cuda_device)
    ids[:, 20:] = padding % 300
    weight = torch.randn(300, 48, device=cuda_device, dtype=BF16).requires_grad_()
    out = E.embedding_lookup(weight, ids, padding_idx=padding)
    assert torch.equal(out, weight.detach()[ids])  # the row itself is looked up like others
    d = torch.randn_like(out)
    (grad,) = torch.autograd.grad(out, weight, d)
    assert not grad[padding % 300].any()
    check_gradient(grad, d, ids, 300, 1.0, padding=padding)


def test_rows_of_any_pitch_and_alignment(cuda_device):
    big = torch.randn(900, 200, device=cuda_device, dtype=BF16)
    ids = torch.randint(0, 300, (77,), device=cuda_device)
    for weight in (big[1::3, 3:120], big[:300, 1:2], big[5:305, :199], big[:300].t().contiguous().t()[:, :1]):
        check_rows(E.embedding_lookup(weight, ids, scale=1.5), weight, ids, 1.5)
    for d in (big[:77, 3:120], big[1:155:2, :64], big[7:8, :33].expand(77, 33), torch.ones((), device=cuda_device).expand(77, 20),
              big.t()[:77, :64], big[:77, :1]):
        check_gradient(E.embedding_backward_accumulate(d, ids, torch.zeros(300, d.shape[1], device=cuda_device)), d, ids, 300, 1.0)


def test_a_broadcast_gradient(cuda_device):
    weight = torch.randn(50, 24, device=cuda_device).requires_grad_()
    ids = torch.randint(0, 50, (6, 9), device=cuda_device, dtype=torch.int32)
    E.embedding_lookup(weight, ids).sum().backward()
    counts = torch.bincount(ids.reshape(-1).long(), minlength=50).float()
    assert torch.equal(weight.grad, counts[:, None].expand(50, 24))


def test_gradient_against_differences(cuda_device):
    """The operator is linear in the table: what a change of the table does to a weighted sum of rows is the gradient's product with it."""
    gen = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 90, (200,), generator=gen).to(cuda_device)
    weight, change = (torch.randint(-8, 9, (90, 40), generator=gen).float().to(cuda_device) for _ in range(2))
    d = torch.randint(-4, 5, (200, 40), generator=gen).float().to(cuda_device)
    (grad,) = torch.autograd.grad(E.embedding_lookup(weight.requires_grad_(), ids, scale=2.0), weight, d)
    with torch.no_grad():
        moved = E.embedding_lookup(weight + change, ids, scale=2.0) - E.embedding_lookup(weight, ids, scale=2.0)
    assert float((moved * d).double().sum()) == float((grad * change).double().sum())  # whole numbers below 2^24: exact


def test_non_finite_values_stay_in_their_rows(cuda_device):
    ids = torch.tensor([3, 1, 3, 2, 1], device=cuda_device)
    d = torch.ones(5, 20, device=cuda_device)
    d[2, 5], d[4, 6] = float("inf"), float("nan")
    grad = E.lmhead_embedding_bwd(d, ids, 6, 1.0, -1)
    want = torch.zeros(6, 20, device=cuda_device)
    want[1], want[2], want[3] = 2.0, 1.0, 2.0
    want[3, 5], want[1, 6] = float("inf"), float("nan")
    assert torch.equal(grad.nan_to_num(7.0), want.nan_to_num(7.0))


def test_empty_inputs(cuda_device):
    weight = torch.randn(10, 8, device=cuda_device).requires_grad_()
    out = E.embedding_lookup(weight, torch.empty((0, 3), dtype=torch.int64, device=cuda_device))
    assert out.shape == (0, 3, 8)
    out.sum().backward()
    assert not weight.grad.any()
    buffer = torch.ones(10, 8, device=cuda_device)
    E.embedding_backward_accumulate(out.detach(), torch.empty((0, 3), dtype=torch.int64, device=cuda_device), buffer)
    assert bool((buffer == 1).all())
    assert E.embedding_lookup(torch.empty(0, 8, device=cuda_device), torch.zeros(4, dtype=torch.int64, device=cuda_device)).abs().max() == 0


def test_replays_from_a_graph_and_on_another_stream(cuda_device):
    T, H, V = 5000, 64, 400
    weight = torch.randn(V, H, device=cuda_device, dtype=BF16)
    ids, d = torch.randint(0, V, (T,), device=cuda_device), torch.randn(T, H, device=cuda_device, dtype=BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        E.lmhead_embedding_bwd(d, ids, V, 1.0, -1)
        E.lmhead_embedding_fwd(weight, ids, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows, grad = E.lmhead_embedding_fwd(weight, ids, 1.0), E.lmhead_embedding_bwd(d, ids, V, 1.0, -1)
    for seed in range(4):
        gen = torch.Generator(device=cuda_device).manual_seed(seed)
        ids.copy_(torch.randint(-1, V, (T,), generator=gen, device=cuda_device))
        d.copy_(torch.randn(T, H, generator=gen, device=cuda_device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(rows, E.lmhead_embedding_fwd(weight, ids, 1.0))
        eager = E.lmhead_embedding_bwd(d, ids, V, 1.0, -1)
        assert torch.equal(grad, eager)
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            other = E.lmhead_embedding_bwd(d, ids, V, 1.0, -1)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, eager)


def test_rows_beyond_32_bit_offsets(cuda_device):
    """A table of 4.6 GB, and its gradient: rows on both sides of 2^31 and 2^32 bytes."""
    V, H = 1_200_000, 1920
    weight = torch.zeros(V, H, dtype=BF16, device=cuda_device)
    ids = torch.tensor([0, 559_240, 559_241, 1_118_480, 1_118_482, V - 1, V], device=cuda_device)
    weight[ids[:-1]] = torch.arange(1, 7, device=cuda_device, dtype=BF16)[:, None]
    out = E.embedding_lookup(weight, ids)
    assert torch.equal(out[:, 7].cpu().float(), torch.tensor([1.0, 2, 3, 4, 5, 6, 0]))
    grad = E.lmhead_embedding_bwd(out, ids, V, 1.0, -1)
    assert torch.equal(grad, weight)


def test_a_second_derivative_is_refused(cuda_device):
    weight = torch.randn(5, 8, device=cuda_device).requires_grad_()
    out = E.embedding_lookup(weight, torch.tensor([1, 2], device=cuda_device))
    up = torch.ones_like(out).requires_grad_()
    (grad,) = torch.autograd.grad(out, weight, up, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_compiled_programs_see_the_ops(cuda_device):
    weight, ids = torch.randn(30, 16, device=cuda_device), torch.tensor([4, 29, 30], device=cuda_device)
    for op, args in ((E.lmhead_embedding_fwd, (weight, ids, 0.5)), (E.lmhead_embedding_bwd, (weight[:3].contiguous(), ids, 30, 0.5, 4))):
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("T,kind", [(65536, "text"), (65537, "text"), (70001, "some outside"), (1100003, "text"), (1100003, "apart"), (1100003, "one")])
def test_more_blocks_than_one_launch_merges(cuda_device, T, kind):
    """Whole numbers, whose sums are exact in fp32 (at most 1.1 million of them, 7 the largest): a token that the sort loses or counts twice shows."""
    gen = torch.Generator().manual_seed(T)
    ids = some_ids(kind, T, 40009, gen).to(cuda_device)
    d = torch.randint(-7, 8, (T, 4), generator=gen).float()
    want, _, _ = plain_gradient(d, ids, 40009, 1.0)
    assert torch.equal(E.lmhead_embedding_bwd(d.to(cuda_device), ids, 40009, 1.0, -1).double().cpu(), want)
