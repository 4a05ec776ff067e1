"""The head in 8-bit integers (``skyrl_amd.int8_head``) against the definitions in 64 bits.

Integers are compared exactly.  Tolerances: a logit is an exact sum, its conversion to fp32, two products and the token's scale: four roundings of 2^-24
(2^-22 relative), and eps / 2 of the type that it is stored in.  In log-probabilities and entropies a logit's relative 2^-22 counts with the largest |z| of
a row; exponentials, sums of V terms over parts of 128 and the merge add at most 2^-24 (64 + |lse|) and are below 1e-5 here; of the entropy, whose terms are products of up to |z|, ten times
that.
"""

from __future__ import annotations

import math

import pytest
import torch

from skyrl_amd import int8_head as I
from skyrl_amd import torch_utils as TU

pytestmark = pytest.mark.gpu
BF16, F32, NAN = torch.bfloat16, torch.float32, math.nan


def plain_integers(x):
    """(q, step) of rows in 64 bits.  Exact: the remainder of 2 * 127 |x| by m says on which side of the border between two integers the quotient lies."""
    x = x.double().cpu()
    m = x.abs().amax(1, keepdim=True)
    low = torch.floor(x.abs() * 127 / m)
    twice = 254.0 * x.abs() - (2 * low + 1) * m  # 8 and 24 bits times 24: exact in 53
    q = (low + ((twice > 0) | ((twice == 0) & (low % 2 == 1))).double()) * x.sign()
    q = torch.where(m > 0, q, 0.0)
    odd = ~torch.isfinite(m)
    return torch.where(odd, 0.0, q), torch.where(odd, NAN, m / 127)


def plain_logits(hidden, head):
    q, step = plain_integers(hidden)
    w = head.values[:, :hidden.shape[1]].double().cpu()
    return (q @ w.T) * step * head.scale.double().cpu()


def some_head(V, H, dtype, gen, device):
    weight = torch.randn(V, H, generator=gen) * 2 / math.sqrt(H)
    return I.quantize_head(weight.to(dtype).to(device))


def some_hidden(T, H, dtype, gen, device):
    x = torch.randn(T, H, generator=gen) * (1 + 6 * (torch.rand(H, generator=gen) < 0.02))
    return x.to(dtype).to(device)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,H", [(1, 1), (3, 7), (5, 8), (2, 127), (40, 128), (9, 129), (300, 896), (7, 4096), (2, 20001)])
def test_integers_of_rows(cuda_device, n, H, dtype):
    gen = torch.Generator().manual_seed(H)
    x = torch.randn(n, H, generator=gen).to(dtype)
    x[0] = 0
    for r in range(1, n):
        x[r] *= 2.0 ** (r % 60 - 30)
    got = I.quantize_head(x.to(cuda_device))
    q, step = plain_integers(x)
    assert got.values.shape == (n, -(-H // 128) * 128) and got.values.dtype == torch.int8 and got.scale.dtype == F32
    assert torch.equal(got.values[:, :H].cpu().double(), q) and not got.values[:, H:].any()
    assert torch.equal(got.scale.cpu(), step[:, 0].float()) or bool(((got.scale.cpu().double() - step[:, 0]).abs() <= 2.0 ** -24 * step[:, 0]).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quotients_exactly_between_integers_go_to_the_even_one(cuda_device, dtype):
    x = torch.zeros(4, 300)
    x[0] = torch.arange(300) - 150.0
    x[0, 0], x[0, 1:255] = 254.0, torch.arange(-127, 127).float()  # 127 x / 254: x / 2
    x[1], x[1, 0] = x[0] * 2.0 ** -100, 254 * 2.0 ** -100
    x[2, :5] = torch.tensor([127.0, 0.5, -0.5, 1.5, 2.5])
    x[3, :4] = torch.tensor([3.0e38, 1.0e38, -2.0e38, 1.18e36])
    got = I.quantize_head(x.to(dtype).to(cuda_device))
    assert torch.equal(got.values[:, :300].cpu().double(), plain_integers(x.to(dtype))[0])
    assert got.values[2, :5].tolist() == [127, 0, 0, 2, 2]


def test_neighbours_of_the_border(cuda_device):
    """fp32 quotients as near to the border between two integers as they get, on both sides."""
    m = torch.arange(2 ** 24 - 40, 2 ** 24, dtype=torch.float64).repeat_interleave(64)
    k = (torch.arange(64, dtype=torch.float64) * 2 + 1).repeat(40)
    near = torch.round(m * k / 254)
    x = torch.stack([torch.stack([m[i], near[i] - 1, near[i], near[i] + 1]) for i in range(len(m))]).float()
    got = I.quantize_head(x.to(cuda_device))
    assert torch.equal(got.values[:, :4].cpu().double(), plain_integers(x)[0])


def test_rows_with_nan_or_infinities(cuda_device):
    x = torch.randn(5, 200)
    x[1, 3], x[2, 4], x[3, 5] = NAN, math.inf, -math.inf
    got = I.quantize_head(x.to(cuda_device))
    assert got.scale.isnan().tolist() == [False, True, True, True, False] and not got.values[1:4].any()
    assert torch.equal(got.values[[0, 4], :200].cpu().double(), plain_integers(x[[0, 4]])[0])


SIZES = [(1, 64, 1), (1, 128, 300), (3, 1, 5), (16, 896, 1000), (17, 200, 4099), (33, 1536, 999), (64, 129, 513), (100, 384, 257), (128, 257, 2000), (129, 256, 2001),
         (137, 896, 1537), (200, 640, 129), (300, 128, 5003), (513, 512, 700), (700, 1023, 300)]


@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("T,H,V", SIZES)
def test_logits(cuda_device, T, H, V, dtype, out):
    gen = torch.Generator().manual_seed(T + H + V)
    head, hidden = some_head(V, H, dtype, gen, cuda_device), some_hidden(T, H, dtype, gen, cuda_device)
    got = I.int8_logits(hidden, head, dtype=out)
    want = plain_logits(hidden, head)
    assert got.dtype == out and got.shape == (T, V)
    bound = want.abs() * (2.0 ** -22 + torch.finfo(out).eps / 2 * 1.001) + 1e-30
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), (off - bound).max()


@pytest.mark.parametrize("temperature", [1.0, 0.6])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,H,V", SIZES + [(2, 3584, 20011)])
def test_logprobs(cuda_device, T, H, V, dtype, temperature):
    gen = torch.Generator().manual_seed(T + H + V)
    head, hidden = some_head(V, H, dtype, gen, cuda_device), some_hidden(T, H, dtype, gen, cuda_device)
    labels = torch.randint(0, V, (T,), generator=gen)
    labels[T // 3::7] = -100
    labels[T // 2::9] = V
    lp, ent = I.int8_logprobs_from_hidden(hidden, head, labels.to(cuda_device), temperature=temperature)
    check_logprobs(lp, ent, plain_logits(hidden, head) / temperature, labels)
    alone, none = I.int8_logprobs_from_hidden(hidden, head, labels.to(cuda_device), temperature=temperature, compute_entropy=False)
    assert torch.equal(alone, lp) and none.numel() == 0


def check_logprobs(lp, ent, y, labels):
    V = y.shape[1]
    logp = torch.log_softmax(y, 1)
    has = (labels >= 0) & (labels < V)
    want = torch.where(has, logp.gather(1, torch.where(has, labels, 0)[:, None])[:, 0], 0.0)
    entropy = -(logp.exp() * logp).sum(1)
    unit = 2.0 ** -22 * y.abs().amax(1) * 2 + 1e-5
    assert lp.dtype == ent.dtype == F32
    assert bool(((lp.double().cpu() - want).abs() <= unit).all()), (lp.double().cpu() - want).abs().max()
    assert bool(((ent.double().cpu() - entropy).abs() <= 10 * unit).all()), (ent.double().cpu() - entropy).abs().max()
    assert bool((lp[~has.to(lp.device)] == 0).all())


def test_the_largest_sums_are_exact(cuda_device):
    """All values +-127 at the largest hidden size: a sum of 2^31 - 2^14 and more."""
    H = I.MAX_HIDDEN
    head = I.Int8Head(torch.full((130, H), 127, dtype=torch.int8, device=cuda_device), torch.ones(130, device=cuda_device))
    head.values[1] = -127
    head.values[2, ::2] = -127
    for T in (1, 130):
        hidden = torch.ones(T, H, device=cuda_device)
        z = I.int8_logits(hidden, head, dtype=F32)
        want = 127.0 * H
        assert want * 127 < 2 ** 31
        got = z[0, :3].double().cpu()
        assert abs(got[0] - want) <= want * 2 ** -22 and abs(got[1] + want) <= want * 2 ** -22 and got[2] == 0
        assert torch.equal(z, z[:1].expand_as(z))


@pytest.mark.parametrize("T", [1, 40, 130])
def test_the_largest_sums_of_a_weight_of_minus_128(cuda_device, T):
    """-128, which quantize_head does not make, at the largest hidden size: a sum of 127 * 128 * H, on either side of zero."""
    H = I.MAX_HIDDEN
    assert 127 * 128 * H < 2 ** 31 <= 127 * 128 * (H + 128)
    head = I.Int8Head(torch.full((70, H), -128, dtype=torch.int8, device=cuda_device), torch.ones(70, device=cuda_device))
    hidden = torch.ones(T, H, device=cuda_device)
    hidden[T // 2:] = -1
    z = I.int8_logits(hidden, head, dtype=F32).double().cpu()
    want = -128.0 * H * hidden[:, :1].double().cpu()
    assert bool(((z - want).abs() <= 128.0 * H * 2 ** -22).all())
    lp, _ = I.int8_logprobs_from_hidden(hidden, head, torch.zeros(T, dtype=torch.int64, device=cuda_device))
    # 70 equal logits; the label's is summed on its own, and both are rounded to fp32 (1.7e7: steps of 1 or 2)
    assert bool(((lp.double().cpu() + math.log(70)).abs() <= 128.0 * H * 2 ** -21).all())


@pytest.mark.parametrize("T", [3, 40, 200])
def test_what_lies_behind_the_hidden_size_does_not_enter(cuda_device, T):
    gen = torch.Generator().manual_seed(1)
    head, hidden = some_head(500, 200, BF16, gen, cuda_device), some_hidden(T, 200, BF16, gen, cuda_device)
    clean = I.int8_logits(hidden, head, dtype=F32)
    room = torch.full((500, 400), 77, dtype=torch.int8, device=cuda_device)  # rows of a wider pitch, anything behind
    room[:, :200] = head.values[:, :200]
    labels = torch.arange(T, device=cuda_device)
    for values in (room[:, :256], room[:, :256].contiguous()):
        assert torch.equal(I.int8_logits(hidden, I.Int8Head(values, head.scale), dtype=F32), clean)
        assert all(torch.equal(a, b) for a, b in zip(I.int8_logprobs_from_hidden(hidden, I.Int8Head(values, head.scale), labels),
                                                     I.int8_logprobs_from_hidden(hidden, head, labels)))


@pytest.mark.parametrize("T", [2, 70, 300])
def test_rows_of_any_pitch_and_scales_of_any_sign(cuda_device, T):
    gen = torch.Generator().manual_seed(2)
    head = some_head(700, 130, BF16, gen, cuda_device)
    scale = torch.cat([torch.zeros(1, device=cuda_device), head.scale])[1:] * torch.where(torch.arange(700, device=cuda_device) % 3 == 0, -1.0, 1.0)
    scale[5] = 0
    signed = I.Int8Head(head.values, scale)
    big = some_hidden(3 * T, 400, BF16, gen, cuda_device)
    for hidden in (big[::3, 3:133], big[:T, 100:230], big[1:2, :130].expand(T, 130), big[:T, :260:2], big.t()[:130, :T].t()):
        want = plain_logits(hidden.contiguous(), signed)
        got = I.int8_logits(hidden, signed, dtype=F32).double().cpu()
        assert bool(((got - want).abs() <= want.abs() * 2.0 ** -22 + 1e-30).all())
        labels = torch.arange(T) % 700
        check_logprobs(*I.int8_logprobs_from_hidden(hidden, signed, labels.to(cuda_device)), want, labels)
    assert I.int8_logits(big[:T, :130].reshape(T, 1, 130), signed).shape == (T, 1, 700)


@pytest.mark.parametrize("T", [4, 60, 260])
def test_odd_rows(cuda_device, T):
    """Hidden rows of zeros, with NaN, with an infinity; a vocabulary row whose scale is NaN."""
    gen = torch.Generator().manual_seed(3)
    head, hidden = some_head(600, 256, BF16, gen, cuda_device), some_hidden(T, 256, BF16, gen, cuda_device)
    hidden[0], hidden[1, 9], hidden[2, 200] = 0, NAN, math.inf
    labels = torch.arange(T)
    z = I.int8_logits(hidden, head, dtype=F32)
    assert not z[0].any() and z[1:3].isnan().all() and not z[3:].isnan().any()
    lp, ent = I.int8_logprobs_from_hidden(hidden, head, labels.to(cuda_device))
    assert lp[1:3].isnan().all() and ent[1:3].isnan().all()
    assert abs(float(lp[0]) + math.log(600)) < 1e-5 and abs(float(ent[0]) - math.log(600)) < 1e-5
    keep = [0, *range(3, T)]
    check_logprobs(lp[keep], ent[keep], plain_logits(hidden[keep], head), labels[keep])
    head.scale[77] = NAN
    z = I.int8_logits(hidden[3:], head)
    assert z[:, 77].isnan().all() and not z[:, :77].isnan().any() and not z[:, 78:].isnan().any()
    assert I.int8_logprobs_from_hidden(hidden[3:], head, labels[3:].to(cuda_device))[0].isnan().all()


def test_far_logits(cuda_device):
    """Rows whose probabilities are all on one token, and logits around +-1e5."""
    gen = torch.Generator().manual_seed(4)
    head = some_head(3000, 128, BF16, gen, cuda_device)
    hidden = some_hidden(140, 128, F32, gen, cuda_device) * torch.logspace(-3, 4, 140, device=cuda_device)[:, None]
    y = plain_logits(hidden, head)
    labels = y.argmax(1)
    check_logprobs(*I.int8_logprobs_from_hidden(hidden, head, labels.to(cuda_device)), y, labels)


def test_more_tokens_than_a_block(cuda_device):
    gen = torch.Generator().manual_seed(6)
    T = 32768 + 300
    head, hidden = some_head(300, 64, BF16, gen, cuda_device), some_hidden(T, 64, BF16, gen, cuda_device)
    labels = torch.randint(0, 300, (T,), generator=gen)
    y = plain_logits(hidden, head)
    check_logprobs(*I.int8_logprobs_from_hidden(hidden, head, labels.to(cuda_device)), y, labels)
    got = I.int8_logits(hidden, head, dtype=F32).double().cpu()
    assert bool(((got - y).abs() <= y.abs() * 2.0 ** -22 + 1e-30).all())


def test_logits_beyond_32_bit_offsets(cuda_device):
    """Logits of 9 GB and values of 5 GB."""
    V, H = 4_700_000, 1024
    values = torch.zeros(V, H, dtype=torch.int8, device=cuda_device)
    at = torch.tensor([0, V // 2, 4_194_304, V - 1], device=cuda_device)
    values[at, 0] = torch.tensor([1, 2, 3, 4], dtype=torch.int8, device=cuda_device)
    head = I.Int8Head(values, torch.ones(V, device=cuda_device))
    for T in (5, 500):
        hidden = torch.zeros(T, H, device=cuda_device, dtype=BF16)
        hidden[:, 0] = 127
        z = I.int8_logits(hidden, head)
        assert z[T - 1, at].tolist() == [127, 254, 381, 508] or torch.equal(z[T - 1, at].float().cpu(), torch.tensor([127.0, 254, 381, 508]).bfloat16().float())
        assert int((z[T - 1] != 0).sum()) == 4
        lp, _ = I.int8_logprobs_from_hidden(hidden * 1e-3, head, at[:1].expand(T).contiguous())
        assert torch.isfinite(lp).all()


def test_replays_from_a_graph_and_on_another_stream(cuda_device):
    gen = torch.Generator().manual_seed(7)
    head, hidden = some_head(5000, 384, BF16, gen, cuda_device), some_hidden(40, 384, BF16, gen, cuda_device)
    labels = torch.randint(0, 5000, (40,), generator=gen).to(cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        I.int8_logits(hidden, head), I.int8_logprobs_from_hidden(hidden, head, labels)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z, (lp, ent) = I.int8_logits(hidden, head), I.int8_logprobs_from_hidden(hidden, head, labels)
    for seed in range(3):
        hidden.copy_(some_hidden(40, 384, BF16, torch.Generator().manual_seed(seed), cuda_device))
        graph.replay()
        torch.cuda.synchronize()
        z2, (lp2, ent2) = I.int8_logits(hidden, head), I.int8_logprobs_from_hidden(hidden, head, labels)
        assert torch.equal(z, z2) and torch.equal(lp, lp2) and torch.equal(ent, ent2)
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            z3 = I.int8_logits(hidden, head)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(z3, z2)


def test_logits_and_logprobs_are_of_one_head(cuda_device):
    gen = torch.Generator().manual_seed(8)
    head, hidden = some_head(9001, 896, BF16, gen, cuda_device), some_hidden(150, 896, BF16, gen, cuda_device)
    labels = torch.randint(0, 9001, (150,), generator=gen).to(cuda_device)
    z = I.int8_logits(hidden, head, dtype=F32)
    lp, ent = I.int8_logprobs_from_hidden(hidden, head, labels)
    top = TU.top_logprobs_from_logits(z, labels, 3)
    assert float((top.logprobs - lp).abs().max()) < 2e-5 and float((top.entropy - ent).abs().max()) < 2e-4


def test_no_tokens_and_compiled_programs(cuda_device):
    gen = torch.Generator().manual_seed(9)
    head = some_head(100, 64, BF16, gen, cuda_device)
    empty = torch.empty(0, 5, 64, dtype=BF16, device=cuda_device)
    assert I.int8_logits(empty, head).shape == (0, 5, 100)
    lp, ent = I.int8_logprobs_from_hidden(empty, head, torch.empty(0, 5, dtype=torch.int64, device=cuda_device))
    assert lp.shape == ent.shape == (0, 5)
    hidden, labels = torch.randn(3, 64, device=cuda_device), torch.tensor([0, 1, 2], device=cuda_device)
    for op, args in ((I.lmhead_int8_rows, (hidden,)), (I.lmhead_int8_logits, (hidden, *head, True)), (I.lmhead_int8_fwd, (hidden, *head, labels, 1.0, True))):
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))
