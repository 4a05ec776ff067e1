"""Log-probabilities, ranks, entropy and best alternatives from logits (skyrl_logits_top_fwd / _bwd, ``top_logprobs_from_logits``) against
a plain implementation in 64 bits on the same bf16 / fp32 logits.

Order (ranks and columns) is compared exactly.  Tolerances: a log-probability is ln 2 * (y2 - m) - ln s in fp32 with values up to 2^5:
four roundings of 2^-24 relative to at most 40, and the sum s of V terms accumulated by 512 threads (V / 512 + 20 additions of 2^-24
relative to s): (4 * 40 + V / 512 + 20) * 2^-24 < 5e-5.  The entropy has the same sums, and products of up to 60: below 1e-4 absolute.
Gradients: p has the relative error of its exponent, 2^-24 * 64, and the result one rounding of half an ulp: eps / 2 + 2e-5
relative to the value, and 2e-5 of the largest coefficient for terms that cancel.
"""

from __future__ import annotations

import math

import pytest
import torch

from skyrl_amd import torch_utils as TU

pytestmark = pytest.mark.gpu
INF = math.inf


def plain(logits, labels, k, temperature):
    """The definitions, 64 bits, on the CPU."""
    z = logits.double().cpu() + 0.0
    T, V = z.shape
    nan = torch.isnan(z)
    order = torch.sort(torch.where(nan, -INF, z), dim=1, descending=True, stable=True).indices
    # NaN behind -inf: a second stable pass on whether a column is NaN
    order = order.gather(1, torch.sort(nan.gather(1, order).to(torch.int8), dim=1, stable=True).indices)
    place = torch.empty_like(order).scatter_(1, order, torch.arange(V).expand(T, V).contiguous())
    y = z / temperature
    empty = (z == -INF).all(1)
    lse = torch.logsumexp(y, 1)
    p = torch.exp(y - torch.where(empty, 0.0, lse)[:, None])
    entropy = -(torch.where(p > 0, y - lse[:, None], 0.0) * p).sum(1)
    entropy = torch.where(torch.isnan(lse), lse, entropy)
    ids = order[:, :k].contiguous()
    top = torch.where(empty[:, None], -INF, y.gather(1, ids) - lse[:, None])
    has = (labels >= 0) & (labels < V)
    safe = torch.where(has, labels, 0)[:, None]
    lp = torch.where(has, torch.where(empty, -INF, y.gather(1, safe)[:, 0] - lse), 0.0)
    ranks = torch.where(has & ~nan.gather(1, safe)[:, 0], place.gather(1, safe)[:, 0] + 1, 0)
    return dict(logprobs=lp, entropy=torch.where(empty, 0.0, entropy), ranks=ranks, top_logprobs=top, top_ids=ids, p=torch.where(empty[:, None], 0.0, p),
                y=y, lse=lse, has=has, empty=empty)


def plain_grad(logits, labels, k, temperature, g, q, h):
    w = plain(logits, labels, k, temperature)
    rows = torch.arange(logits.shape[0])
    d = torch.zeros_like(w["p"])
    if g is not None:
        g = torch.where(w["has"], g.double(), 0.0)
        d -= g[:, None] * w["p"]
        d[rows, torch.where(w["has"], labels, 0)] += g
    if q is not None:
        logp = torch.where(w["p"] > 0, w["y"] - w["lse"][:, None], 0.0)
        d -= q.double()[:, None] * w["p"] * (logp + w["entropy"][:, None])
    if h is not None:
        d -= h.double().sum(1, keepdim=True) * w["p"]
        d.scatter_add_(1, w["top_ids"], h.double())
    return torch.where(w["empty"][:, None], 0.0, d / temperature)


def close(got, want, tol):
    got, want = got.detach().cpu().double(), want.double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    assert bool(((got - want).abs().nan_to_num(INF) <= tol).logical_or(same).all()), (got - want).abs().nan_to_num(0.0).max()


def check(logits, labels, k, temperature, device):
    got = TU.top_logprobs_from_logits(logits.to(device), labels.to(device), k, temperature=temperature)
    want = plain(logits, labels, min(k, logits.shape[1]), temperature)
    assert torch.equal(got.top_ids.cpu(), want["top_ids"])
    assert torch.equal(got.ranks.cpu(), want["ranks"])
    close(got.logprobs, want["logprobs"], 5e-5)
    close(got.top_logprobs, want["top_logprobs"], 5e-5)
    close(got.entropy, want["entropy"], 1e-4)
    return got, want


def make(T, V, dtype, seed, scale=2.5):
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn(T, V, generator=gen) * scale).to(dtype)
    labels = torch.randint(0, V, (T,), generator=gen)
    return logits, labels, gen


SIZES = [
    (1, 1, 1, torch.float32), (1, 1, 5, torch.bfloat16), (3, 2, 0, torch.bfloat16), (64, 7, 7, torch.float32), (5, 129, 128, torch.bfloat16),
    (3, 511, 20, torch.float32), (4, 4095, 64, torch.bfloat16), (2, 16384, 33, torch.bfloat16), (2, 16385, 1, torch.float32),
    (17, 20011, 20, torch.bfloat16), (1, 151936, 20, torch.bfloat16), (9, 152064, 128, torch.float32), (300, 32001, 5, torch.bfloat16),
    (1, 600000, 40, torch.bfloat16), (40, 50021, 128, torch.bfloat16), (255, 49152, 3, torch.float32), (257, 49999, 20, torch.bfloat16),
]


@pytest.mark.parametrize("T,V,k,dtype", SIZES)
def test_against_64_bits(T, V, k, dtype, cuda_device):
    logits, labels, _ = make(T, V, dtype, T + V + k)
    labels[::4] = logits[::4].float().argmax(1)  # ranks 1 among them
    if T > 4:
        labels[1], labels[2], labels[3] = -100, V, 2**40
    for temperature in (1.0, 0.3):
        check(logits, labels, k, temperature, cuda_device)


@pytest.mark.parametrize("k", [1, 20, 128])
@pytest.mark.parametrize("kind", ["constant", "ascending", "descending", "few values", "zeros of both signs", "all but one masked", "masked",
                                  "fewer than k", "empty", "nan", "nan and masked", "all nan", "huge", "one huge"])
@pytest.mark.parametrize("V", [33001, 66001])  # a workgroup for a row; eight of them, and their join
def test_rows_that_select_badly(kind, k, V, cuda_device):
    T = 6
    logits, labels, gen = make(T, V, torch.float32, 5)
    ramp = torch.arange(V, dtype=torch.float32) / 1000
    if kind == "constant":
        logits[:] = 1.5
    elif kind == "ascending":
        logits[:] = ramp
    elif kind == "descending":
        logits[:] = -ramp
    elif kind == "few values":
        logits = torch.randint(0, 3, (T, V), generator=gen).float()
    elif kind == "zeros of both signs":
        logits = torch.where(torch.rand(T, V, generator=gen) < 0.5, 0.0, -0.0)
    elif kind == "all but one masked":
        keep = logits.gather(1, labels[:, None])
        logits[:] = -INF
        logits.scatter_(1, labels[:, None], keep)
    elif kind == "masked":
        logits[torch.rand(T, V, generator=gen) < 0.99] = -INF
    elif kind == "fewer than k":
        logits[:, :V - 3] = -INF
    elif kind == "empty":
        logits[::2] = -INF
    elif kind == "nan":
        logits[::2, 7::5] = math.nan
    elif kind == "nan and masked":
        logits[:] = -INF
        logits[:, 5:] = math.nan
        logits[1:, 9] = 2.0
    elif kind == "all nan":
        logits[:] = math.nan
    elif kind == "huge":
        logits *= 1e30
        logits[:, 11] = 3e37
    elif kind == "one huge":
        logits[:, 30000] = 1e6
    for dtype in (torch.float32, torch.bfloat16):
        rows = logits.to(dtype)
        got = TU.top_logprobs_from_logits(rows.to(cuda_device), labels.to(cuda_device), k)
        want = plain(rows, labels, k, 1.0)
        assert torch.equal(got.top_ids.cpu(), want["top_ids"]) and torch.equal(got.ranks.cpu(), want["ranks"])
        if kind == "huge":  # beside a spread of 1e37 only the largest has a probability: the others' log-probabilities lose their low bits
            rel = (got.top_logprobs.cpu().double() - want["top_logprobs"]).abs() / want["top_logprobs"].abs().clamp_min(1.0)
            assert bool((rel.nan_to_num(0.0) <= 2e-6).all())
        else:
            scale = 1e6 if kind == "one huge" else 1.0  # 2^-22 of the largest difference: four roundings
            close(got.top_logprobs, want["top_logprobs"], 5e-5 + scale * 2.0**-22)
            close(got.logprobs, want["logprobs"], 5e-5 + scale * 2.0**-22)
            close(got.entropy, want["entropy"], 1e-4)


@pytest.mark.parametrize("T,V,k,dtype", [(1, 1, 1, torch.float32), (5, 300, 20, torch.bfloat16), (7, 20011, 128, torch.bfloat16),
                                         (3, 151936, 32, torch.bfloat16), (4, 4096, 5, torch.float32), (2, 33, 0, torch.float32)])
@pytest.mark.parametrize("which", ["g", "q", "h", "gqh"])
def test_gradients_against_64_bits(T, V, k, dtype, which, cuda_device):
    logits, labels, gen = make(T, V, dtype, 3 * T + V + k)
    if T > 2:
        labels[0], labels[1] = -1, int(logits[1].float().argmax())  # the label among the alternatives
        logits[2, : V // 2] = -INF
    g = torch.randn(T, generator=gen) if "g" in which else None
    q = torch.randn(T, generator=gen) * 0.1 if "q" in which else None
    h = torch.randn(T, k, generator=gen) if "h" in which and k else None
    if g is None and q is None and h is None:
        return
    temperature = 0.7
    d = logits.to(cuda_device).requires_grad_()
    r = TU.top_logprobs_from_logits(d, labels.to(cuda_device), k, temperature=temperature)
    loss = sum((o * w.to(cuda_device)).sum() for o, w in ((r.logprobs, g), (r.entropy, q), (r.top_logprobs, h)) if w is not None
               for o, w in [(torch.where(torch.isfinite(o), o, 0.0), w)])
    loss.backward()
    h_used = None if h is None else torch.where(torch.isfinite(r.top_logprobs.detach().cpu()), h, 0.0)
    g_used = None if g is None else torch.where(torch.isfinite(r.logprobs.detach().cpu()), g, 0.0)
    want = plain_grad(logits, labels, k, temperature, g_used, q, h_used)
    coefficient = sum(w.double().abs().reshape(T, -1).sum(1) for w in (g_used, h_used) if w is not None) if g is not None or h is not None else torch.zeros(T)
    coefficient = (coefficient + (0 if q is None else 40 * q.double().abs())) / temperature
    err = (d.grad.cpu().double() - want).abs()
    bound = want.abs() * (torch.finfo(dtype).eps / 2 + 2e-5) + 2e-5 * coefficient[:, None] * plain(logits, labels, k, temperature)["p"] + 1e-30
    one_hot = torch.zeros_like(want)  # the columns with a term of their own: that term and the rest may cancel
    one_hot[torch.arange(T), labels.clamp(0)] = 1.0
    one_hot.scatter_(1, plain(logits, labels, k, temperature)["top_ids"], 1.0)
    bound += 2e-6 * coefficient[:, None] * one_hot
    assert d.grad.dtype == dtype and bool((err <= bound).all()), (err - bound).max()


def test_gradient_is_the_difference_quotient(cuda_device):
    logits, labels, gen = make(3, 200, torch.float32, 11, scale=1.0)
    w = [torch.randn(3, generator=gen), torch.randn(3, generator=gen), torch.randn(3, 6, generator=gen)]

    def loss(x):  # 64 bits
        r = plain(x, labels, 6, 0.8)
        return (r["logprobs"] * w[0]).sum() + (r["entropy"] * w[1]).sum() + (r["top_logprobs"] * w[2]).sum()

    d = logits.to(cuda_device).requires_grad_()
    r = TU.top_logprobs_from_logits(d, labels.to(cuda_device), 6, temperature=0.8)
    ((r.logprobs * w[0].to(cuda_device)).sum() + (r.entropy * w[1].to(cuda_device)).sum() + (r.top_logprobs * w[2].to(cuda_device)).sum()).backward()
    step = 1e-5
    for row, col in ((0, 0), (1, int(labels[1])), (2, int(r.top_ids[2, 0])), (0, 199)):
        up, down = logits.double(), logits.double()
        up[row, col] += step
        down[row, col] -= step
        quotient = (loss(up) - loss(down)) / (2 * step)
        assert abs(float(d.grad[row, col]) - float(quotient)) <= 1e-4 * (1 + abs(float(quotient)))


def test_empty_rows_have_no_gradient_and_no_labels_give_no_logprobs(cuda_device):
    logits, labels, _ = make(4, 1000, torch.bfloat16, 2)
    logits[1] = -INF
    d = logits.to(cuda_device).requires_grad_()
    r = TU.top_logprobs_from_logits(d, labels.to(cuda_device), 3)
    (grad,) = torch.autograd.grad((r.logprobs, r.entropy, r.top_logprobs), d, tuple(torch.ones_like(o) for o in (r.logprobs, r.entropy, r.top_logprobs)))
    assert bool((grad[1] == 0).all()) and bool(torch.isfinite(grad).all()) and float(r.logprobs[1].detach()) == -INF
    r = TU.top_logprobs_from_logits(d, None, 3)
    assert not r.logprobs.any() and not r.ranks.any() and r.top_ids.shape == (4, 3)
    (r.entropy.sum() + r.logprobs.sum()).backward()
    assert d.grad is not None


def test_layouts(cuda_device):
    """A slice of a batch, odd pitches, an unaligned start, another dtype, an empty batch; the rows around are left as they are."""
    gen = torch.Generator().manual_seed(1)
    full = (torch.randn(3, 9, 1003, generator=gen) * 2).to(torch.bfloat16).to(cuda_device)
    labels = torch.randint(0, 1000, (3, 8), generator=gen)
    view = full[:, :-1, 2:1002].requires_grad_()
    r = TU.top_logprobs_from_logits(view, labels.to(cuda_device), 4)
    want = plain(view.detach().reshape(-1, 1000).cpu(), labels.reshape(-1), 4, 1.0)
    assert r.top_ids.shape == (3, 8, 4) and torch.equal(r.top_ids.reshape(-1, 4).cpu(), want["top_ids"])
    close(r.logprobs.reshape(-1), want["logprobs"], 5e-5)
    (grad,) = torch.autograd.grad(r.top_logprobs.sum(), view)
    close(grad.reshape(-1, 1000), plain_grad(view.detach().reshape(-1, 1000).cpu(), labels.reshape(-1), 4, 1.0, None, None, torch.ones(24, 4)), 2.0**-8)
    half = TU.top_logprobs_from_logits(full[0, :, :64].half(), labels[0, :1].expand(9).to(cuda_device) % 64, 2)
    assert torch.equal(half.top_ids.cpu(), plain(full[0, :, :64].half().cpu(), torch.zeros(9, dtype=torch.int64), 2, 1.0)["top_ids"])
    none = TU.top_logprobs_from_logits(full[:0, 0], labels[:0, 0].to(cuda_device), 4)
    assert none.logprobs.shape == (0,) and none.top_ids.shape == (0, 4)


def test_same_bits_on_each_call_and_on_another_stream(cuda_device):
    logits, labels, _ = make(8, 151936, torch.bfloat16, 4)
    d, y = logits.to(cuda_device), labels.to(cuda_device)
    first = TU.top_logprobs_from_logits(d, y, 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = TU.top_logprobs_from_logits(d, y, 20)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    for T, V, dtype in ((64, 151936, torch.float32), (1500, 30000, torch.bfloat16)):
        logits, labels, _ = make(T, V, dtype, 4)
        d, y = logits.to(cuda_device), labels.to(cuda_device)
        first = TU.top_logprobs_from_logits(d, y, 20)
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(first, TU.top_logprobs_from_logits(d, y, 20)))


@pytest.mark.parametrize("V", [30001, 70001])
def test_replays_from_a_graph(V, cuda_device):
    gen = torch.Generator().manual_seed(9)
    d = torch.zeros(5, V, dtype=torch.bfloat16, device=cuda_device)
    y = torch.zeros(5, dtype=torch.int64, device=cuda_device)
    h = torch.rand(5, 7, generator=gen).to(cuda_device)

    def step():
        with torch.no_grad():
            lp, ent, lse, pz, ranks, top, ids = TU.logits_top_fwd(d, y, 7, 1.25)
            return lp, ent, ranks, top, ids, TU.logits_top_bwd(d, y, lse, pz, lp, ent, ids, h, 1.25)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        logits, labels, _ = make(5, V, torch.bfloat16, 100 + i)
        d.copy_(logits)
        y.copy_(labels)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals_of_the_python_entry_point(cuda_device):
    z, y = torch.zeros(2, 50, device=cuda_device), torch.zeros(2, dtype=torch.int64, device=cuda_device)
    for bad in (lambda: TU.top_logprobs_from_logits(z, y, 129), lambda: TU.top_logprobs_from_logits(z, y, -1), lambda: TU.top_logprobs_from_logits(z, y, 2.0),
                lambda: TU.top_logprobs_from_logits(z, y[:1], 2), lambda: TU.top_logprobs_from_logits(z, y, 2, temperature=0.0),
                lambda: TU.top_logprobs_from_logits(z, y, 2, temperature=math.nan), lambda: TU.logits_top_fwd(z, y, 51, 1.0)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        TU.top_logprobs_from_logits(z.cpu(), y.cpu(), 2)
    assert TU.top_logprobs_from_logits(z, y, 128).top_ids.shape == (2, 50)
