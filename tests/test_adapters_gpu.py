"""The head with adapters of many requests (``skyrl_amd.adapters``) against a plain implementation in 64 bits on the same bf16 operands.

Tolerances, with e = 2^-8 for a rounding to bf16 (half a step).  A logit is a sum of H + 2 R products that are exact in fp32: its error is below
(H + 2 R) * 2^-24 * sum |terms|, and u as two bf16 terms adds 2^-16 * sum |u B|; call it z_err.  Log-probability and entropy: the logit's and
the log-sum-exp's error, z_err each, the entropy's twice over because p z is weighted, and 5e-5 for the sums over V.  Gradients: dz is rounded
once (e), u once more in dB (e), each result once (e), d_hidden twice (2 e); p carries a relative error of 2 z_err.  The roundings of the
many terms of a sum are independent, so that a result's norm is off by at most 3 e + 2 z_err of its norm; norms are taken row by row (a token's
d_hidden, an adapter's dA and dB), so that no row hides in another.
"""

from __future__ import annotations

import math

import pytest
import torch

from skyrl_amd import ops
from skyrl_amd import adapters as AD
from skyrl_amd import torch_utils as TU

pytestmark = pytest.mark.gpu
E = 2.0**-8


def make(T, H, V, N, R, order="runs", seed=0, b_scale=0.08):
    gen = torch.Generator().manual_seed(seed)
    b16 = torch.bfloat16
    hidden = torch.randn(T, H, generator=gen).to(b16)
    weight = (torch.randn(V, H, generator=gen) * (2.0 / math.sqrt(H))).to(b16)
    a = (torch.randn(N, R, H, generator=gen) / math.sqrt(H)).to(b16)
    b = (torch.randn(N, V, R, generator=gen) * b_scale).to(b16)
    scaling = 0.5 + 1.5 * torch.rand(N, generator=gen)
    if order == "one":
        ids = torch.full((T,), N - 1)
    elif order == "mixed":
        ids = torch.randint(-1, N, (T,), generator=gen)
    else:
        cuts = torch.sort(torch.randint(0, T + 1, (2 * N + 1,), generator=gen)).values
        ids = torch.randint(-1, N, (2 * N + 2,), generator=gen)[torch.bucketize(torch.arange(T), cuts, right=True)]
    return hidden, weight, a, b, scaling, ids, gen


def plain_logits(hidden, weight, a, b, scaling, ids):
    """64 bits, differentiable; token by token where it matters: no token sees another's adapter."""
    h, w, a, b = (x.double() for x in (hidden, weight, a, b))
    z = h @ w.T
    rows = []
    for n in range(a.shape[0]):
        at = (ids == n).nonzero()[:, 0]
        if at.numel():
            rows.append((at, scaling[n].double() * ((h[at] @ a[n].T) @ b[n].T)))
    for at, more in rows:
        z = z.index_add(0, at, more)
    return z


def z_error(hidden, weight, a, b, scaling, ids):
    h, w, a, b = (x.double().abs() for x in (hidden, weight, a, b))
    T, H = h.shape
    R = a.shape[1]
    err = (H + 2 * R) * 2.0**-24 * (h @ w.T)
    for n in range(a.shape[0]):
        at = (ids == n).nonzero()[:, 0]
        if at.numel():
            err[at] += ((H + 2 * R) * 2.0**-24 + 2.0**-16) * scaling[n].double().abs() * ((h[at] @ a[n].T) @ b[n].T)
    return err


def on(device, *tensors):
    return tuple(t.to(device) for t in tensors)


LOGITS = [
    (1, 64, 1, 1, 8, "one"), (1, 64, 1000, 3, 8, "mixed"), (2, 128, 257, 2, 16, "mixed"), (16, 896, 4099, 8, 16, "mixed"), (17, 192, 5000, 70, 8, "mixed"),
    (128, 256, 3001, 48, 32, "mixed"), (129, 256, 3000, 5, 24, "runs"), (217, 128, 4097, 5, 40, "runs"), (256, 64, 2048, 4, 64, "mixed"),
    (300, 320, 1111, 2, 256, "runs"), (513, 128, 700, 9, 72, "mixed"),
]


@pytest.mark.parametrize("T,H,V,N,R,order", LOGITS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logits_against_64_bits(T, H, V, N, R, order, dtype, cuda_device):
    *x, _ = make(T, H, V, N, R, order, seed=T + V)
    got = AD.adapter_logits(*on(cuda_device, *x), dtype=dtype).cpu()
    want, err = plain_logits(*x), z_error(*x)
    assert got.dtype == dtype and got.shape == (T, V)
    bound = err + (want.abs() * E if dtype == torch.bfloat16 else 0.0)
    assert bool(((got.double() - want).abs() <= bound).all()), ((got.double() - want).abs() - bound).max()


TRAIN = [
    (1, 64, 300, 1, 8, "one", 1.0), (3, 64, 128, 2, 8, "mixed", 1.0), (40, 128, 1000, 3, 16, "mixed", 0.7), (64, 64, 2049, 2, 24, "runs", 1.0),
    (137, 192, 3001, 5, 16, "runs", 1.0), (200, 128, 1024, 70, 8, "mixed", 1.3), (300, 256, 5003, 4, 32, "runs", 0.7), (611, 128, 777, 12, 40, "runs", 1.0),
    (520, 64, 4096, 3, 64, "mixed", 1.0), (140, 320, 1500, 2, 256, "runs", 1.0),
]


def row_norms(got, want, tol, floor):
    """|got - want| <= tol |want| + floor, row by row of the last dimension's blocks."""
    got, want = got.double().cpu().flatten(1), want.double().flatten(1)
    off = (got - want).norm(dim=1)
    assert bool((off <= tol * want.norm(dim=1) + floor).all()), (off / want.norm(dim=1).clamp_min(1e-30)).max()


@pytest.mark.parametrize("T,H,V,N,R,order,temperature", TRAIN)
@pytest.mark.parametrize("entropy_grad", [False, True])
def test_training_against_64_bits(T, H, V, N, R, order, temperature, entropy_grad, cuda_device):
    *x, gen = make(T, H, V, N, R, order, seed=T + V + R)
    labels = torch.randint(0, V, (T,), generator=gen)
    if T > 4:
        labels[1], labels[3] = -100, V
    g, q = torch.randn(T, generator=gen), torch.randn(T, generator=gen) * 0.1
    masked = (torch.rand(T, generator=gen) < 0.3) & (T > 2)
    g[masked], q[masked] = 0.0, 0.0
    leaves = [x[i].double().requires_grad_() for i in (0, 2, 3)]
    z = plain_logits(leaves[0], x[1], leaves[1], leaves[2], x[4], x[5]) / temperature
    lsm = torch.log_softmax(z, 1)
    has = (labels >= 0) & (labels < V)
    want_lp = torch.where(has, lsm.gather(1, labels.clamp(0, V - 1)[:, None])[:, 0], 0.0)
    want_ent = -(lsm.exp() * lsm).sum(1)
    # a label outside the vocabulary keeps -softmax * g in the backward, as in the head without adapters
    loss = (torch.where(has, want_lp, -torch.logsumexp(z, 1)) * g).sum() + ((want_ent * q).sum() if entropy_grad else 0.0)
    want = torch.autograd.grad(loss, leaves)

    d = on(cuda_device, *x)
    dl = [d[i].clone().requires_grad_() for i in (0, 2, 3)]
    lp, ent = AD.adapter_logprobs_from_hidden(dl[0], d[1], labels.to(cuda_device), dl[1], dl[2], d[4], d[5], temperature=temperature)
    z_err = float(z_error(*x).max()) / temperature
    assert float((lp.detach().cpu().double() - want_lp.detach()).abs().max()) <= 2 * z_err + 5e-5
    assert float((ent.detach().cpu().double() - want_ent.detach()).abs().max()) <= 4 * z_err * (1 + math.log(V)) + 5e-5
    back = (lp * g.to(cuda_device)).sum() + ((ent * q.to(cuda_device)).sum() if entropy_grad else 0.0)
    got = torch.autograd.grad(back, dl)
    tol = 3 * E + 2 * z_err
    for name, a, b in zip(("d_hidden", "d_lora_a", "d_lora_b"), got, want):
        assert a.dtype == torch.bfloat16 and a.shape == b.shape, name
        row_norms(a, b, tol, 1e-6 * float(b.norm()) + 1e-12)
    assert not bool(got[0][masked.to(cuda_device)].any())
    unused = [n for n in range(N) if not bool(((x[5] == n) & ~masked).any())]
    assert all(not bool(got[1][n].any()) and not bool(got[2][n].any()) for n in unused)


def test_gradient_is_the_difference_quotient(cuda_device):
    *x, gen = make(20, 64, 150, 2, 8, "mixed", seed=3)
    labels, g, q = torch.randint(0, 150, (20,), generator=gen), torch.randn(20, generator=gen), torch.randn(20, generator=gen)

    def loss(h, a, b):
        z = plain_logits(h, x[1], a, b, x[4], x[5])
        lsm = torch.log_softmax(z, 1)
        return float((lsm.gather(1, labels[:, None])[:, 0] * g).sum() - ((lsm.exp() * lsm).sum(1) * q).sum())

    d = on(cuda_device, *x)
    dl = [d[i].clone().requires_grad_() for i in (0, 2, 3)]
    lp, ent = AD.adapter_logprobs_from_hidden(dl[0], d[1], labels.to(cuda_device), dl[1], dl[2], d[4], d[5])
    got = torch.autograd.grad((lp * g.to(cuda_device)).sum() + (ent * q.to(cuda_device)).sum(), dl)
    base = [x[i].double() for i in (0, 2, 3)]
    for k in range(3):  # along the gradient and along a random direction
        for direction in (got[k].cpu().double(), torch.randn(base[k].shape, generator=gen).double()):
            step = 1e-4 / float(direction.norm())
            up, down = list(base), list(base)
            up[k], down[k] = base[k] + step * direction, base[k] - step * direction
            quotient = (loss(*up) - loss(*down)) / (2 * step)
            along = float((got[k].cpu().double() * direction).sum())
            assert abs(along - quotient) <= 3 * E * float(got[k].double().norm()) * float(direction.norm())


def test_tokens_without_an_adapter_have_the_head_s_own_bits(cuda_device):
    for T in (30, 200, 700):
        *x, gen = make(T, 128, 3000, 3, 16, "mixed", seed=T)
        labels = torch.randint(0, 3000, (T,), generator=gen).to(cuda_device)
        d = on(cuda_device, *x)
        lp, ent, lse, pz = AD.lmhead_adapter_fwd(d[0], d[1], labels, *d[2:], 1.25)
        lp0, ent0, lse0, pz0 = ops.lmhead_fwd(d[0], d[1], labels, 1.25, True)
        none = d[5] < 0
        for a, b in ((lp, lp0), (ent, ent0), (lse, lse0), (pz, pz0)):
            assert torch.equal(a[none], b[none]) and not torch.equal(a[~none], b[~none])
        out = AD.lmhead_adapter_fwd(d[0], d[1], labels, *d[2:5], torch.full_like(d[5], 99), 1.25)
        assert all(torch.equal(a, b) for a, b in zip(out, (lp0, ent0, lse0, pz0)))


@pytest.mark.parametrize("T", [40, 200, 400])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_an_adapter_that_is_not_finite_reaches_its_own_tokens_only(T, bad, cuda_device):
    *x, gen = make(T, 128, 1500, 4, 16, "mixed", seed=T)
    labels = torch.randint(0, 1500, (T,), generator=gen)
    g = torch.randn(T, generator=gen)
    d = on(cuda_device, *x)
    y, gd = labels.to(cuda_device), g.to(cuda_device)
    good = AD.lmhead_adapter_fwd(d[0], d[1], y, *d[2:], 1.0)
    good_grad = AD.lmhead_adapter_bwd(d[0], d[1], y, *d[2:], good[2], None, gd, None, 1.0)
    good_logits = AD.adapter_logits(*d)
    others = d[5] != 2
    for where in ("a", "b", "scaling", "hidden"):
        h, a, b, s = d[0].clone(), d[2].clone(), d[3].clone(), d[4].clone()
        if where == "a":
            a[2, 3, 5] = bad
        elif where == "b":
            b[2, ::7, 4] = bad
        elif where == "scaling":
            s[2] = bad
        else:
            h[d[5] == 2] = bad
        out = AD.lmhead_adapter_fwd(h, d[1], y, a, b, s, d[5], 1.0)
        assert all(torch.equal(p[others], w[others]) for p, w in zip(out, good)), where
        assert not bool(torch.isfinite(out[2][~others]).any()), where
        assert torch.equal(AD.adapter_logits(h, d[1], a, b, s, d[5])[others], good_logits[others])
        grad = AD.lmhead_adapter_bwd(h, d[1], y, a, b, s, d[5], out[2], None, gd, None, 1.0)
        assert torch.equal(grad[0][others], good_grad[0][others]), where
        rest = [0, 1, 3]
        assert torch.equal(grad[1][rest], good_grad[1][rest]) and torch.equal(grad[2][rest], good_grad[2][rest]), where


def test_large_factors_of_shared_blocks(cuda_device):
    """Values of 2 and more in B take the other way through a block of tokens that adapters share."""
    *x, _ = make(100, 128, 900, 6, 16, "mixed", seed=8, b_scale=3.0)
    got = AD.adapter_logits(*on(cuda_device, *x), dtype=torch.float32).cpu()
    assert bool(((got.double() - plain_logits(*x)).abs() <= z_error(*x)).all())


def test_nothing_to_learn_from(cuda_device):
    *x, gen = make(150, 64, 500, 3, 8, "mixed")
    labels = torch.randint(0, 500, (150,), generator=gen)
    d, y = on(cuda_device, *x), labels.to(cuda_device)
    _, _, lse, pz = AD.lmhead_adapter_fwd(d[0], d[1], y, *d[2:], 1.0)
    for grads in (AD.lmhead_adapter_bwd(d[0], d[1], y, *d[2:], lse, pz, torch.zeros_like(lse), None, 1.0),
                  AD.lmhead_adapter_bwd(d[0], d[1], y, *d[2:], lse, pz, torch.zeros_like(lse), torch.zeros_like(lse), 1.0)):
        assert not any(bool(t.any()) for t in grads)
    g = torch.randn(150, generator=gen).to(cuda_device)
    dh, da, db = AD.lmhead_adapter_bwd(d[0], d[1], y, *d[2:5], torch.full_like(d[5], -1), *ops.lmhead_fwd(d[0], d[1], y, 1.0, True)[2:], g, None, 1.0)
    assert not bool(da.any()) and not bool(db.any())
    _, _, lse0, _ = ops.lmhead_fwd(d[0], d[1], y, 1.0, True)
    plain = ops.lmhead_bwd_hidden(d[0], d[1], y, lse0, None, g, None, 1.0, 0, True)
    assert torch.equal(dh, plain)
    empty = AD.adapter_logprobs_from_hidden(d[0][:0].requires_grad_(), d[1], y[:0], d[2].clone().requires_grad_(), d[3], d[4], d[5][:0])
    assert empty[0].shape == (0,)
    empty[0].sum().backward()
    assert AD.adapter_logits(d[0][:0], d[1], *d[2:5], d[5][:0]).shape == (0, 500)


def test_more_tokens_than_one_block(cuda_device):
    T, H, V, N, R = 33100, 64, 260, 3, 8
    *x, gen = make(T, H, V, N, R, "mixed", seed=1)
    labels, g = torch.randint(0, V, (T,), generator=gen), torch.randn(T, generator=gen)
    d, y, gd = on(cuda_device, *x), labels.to(cuda_device), g.to(cuda_device)
    lp, ent, lse, pz = AD.lmhead_adapter_fwd(d[0], d[1], y, *d[2:], 1.0)
    assert torch.equal(lp[:1000], AD.lmhead_adapter_fwd(d[0][:1000], d[1], y[:1000], *d[2:5], d[5][:1000], 1.0)[0]) or \
        float((lp[:1000] - AD.lmhead_adapter_fwd(d[0][:1000], d[1], y[:1000], *d[2:5], d[5][:1000], 1.0)[0]).abs().max()) < 1e-4
    got = AD.lmhead_adapter_bwd(d[0], d[1], y, *d[2:], lse, pz, gd, None, 1.0)
    leaves = [x[i].double().requires_grad_() for i in (0, 2, 3)]
    lsm = torch.log_softmax(plain_logits(leaves[0], x[1], leaves[1], leaves[2], x[4], x[5]), 1)
    want = torch.autograd.grad((lsm.gather(1, labels[:, None])[:, 0] * g).sum(), leaves)
    for a, b in zip(got, want):
        row_norms(a, b, 3 * E + 1e-3, 1e-6 * float(b.norm()))
    logits = AD.adapter_logits(*d)
    assert bool(((logits[32000:].cpu().double() - plain_logits(*x)[32000:]).abs() <= z_error(*x)[32000:] + 0.05).all())


def test_layouts(cuda_device):
    """Operands inside larger ones, a batch of sequences, int32 ids, a stack made of unlike ranks."""
    *x, gen = make(60, 128, 1000, 4, 16, "mixed", seed=4)
    labels = torch.randint(0, 1000, (60,), generator=gen)
    d, y = on(cuda_device, *x), labels.to(cuda_device)
    want = AD.adapter_logprobs_from_hidden(d[0], d[1], y, *d[2:])
    wide = torch.full((60, 200), 7.0, dtype=torch.bfloat16, device=cuda_device)
    wide[:, 8:136] = d[0]
    rows = torch.zeros((1000, 136), dtype=torch.bfloat16, device=cuda_device)
    rows[:, :128] = d[1]
    a = torch.full((9, 24, 136), math.nan, dtype=torch.bfloat16, device=cuda_device)
    b = torch.full((9, 1003, 24), math.nan, dtype=torch.bfloat16, device=cuda_device)
    a[1::2, :16, 8:] = d[2]
    b[1::2, 2:1002, 8:] = d[3]
    got = AD.adapter_logprobs_from_hidden(wide[:, 8:136].view(4, 15, 128), rows[:, :128], y.view(4, 15), a[1::2, :16, 8:], b[1::2, 2:1002, 8:], d[4],
                                          d[5].view(4, 15).to(torch.int32))
    assert got[0].shape == (4, 15) and all(torch.equal(p.reshape(-1), w) for p, w in zip(got, want))
    pairs = [(d[2][n, :r], d[3][n, :, :r]) for n, r in enumerate((16, 5, 8, 1))]
    la, lb, s = AD.stack_adapters(pairs, [1.0, 2.0, 0.5, 1.0])
    assert la.shape == (4, 16, 128) and lb.shape == (4, 1000, 16)
    z = AD.adapter_logits(d[0], d[1], la, lb, s, d[5], dtype=torch.float32)
    cpu = (x[0], x[1], la.cpu(), lb.cpu(), s.cpu(), x[5])
    assert bool(((z.cpu().double() - plain_logits(*cpu)).abs() <= z_error(*cpu)).all())


def test_same_bits_on_each_call_and_on_another_stream(cuda_device):
    *x, gen = make(400, 128, 5000, 5, 16, "mixed", seed=6)
    labels, g = torch.randint(0, 5000, (400,), generator=gen).to(cuda_device), torch.randn(400, generator=gen).to(cuda_device)
    d = on(cuda_device, *x)

    def step():
        lp, ent, lse, pz = AD.lmhead_adapter_fwd(d[0], d[1], labels, *d[2:], 1.0)
        return (lp, ent, AD.adapter_logits(*d)) + AD.lmhead_adapter_bwd(d[0], d[1], labels, *d[2:], lse, pz, g, g, 1.0)

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_replays_from_a_graph(cuda_device):
    T, V = 150, 3000
    d = [t.clone() for t in on(cuda_device, *make(T, 128, V, 3, 16, "mixed", seed=0)[:6])]
    labels, g = torch.zeros(T, dtype=torch.int64, device=cuda_device), torch.zeros(T, device=cuda_device)

    def step():
        lp, ent, lse, pz = AD.lmhead_adapter_fwd(d[0], d[1], labels, *d[2:], 1.0)
        top = TU.logits_top_fwd(AD.lmhead_adapter_logits(*d, False), labels, 5, 1.0)
        return (lp, ent) + tuple(top) + AD.lmhead_adapter_bwd(d[0], d[1], labels, *d[2:], lse, pz, g, None, 1.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        *x, gen = make(T, 128, V, 3, 16, "runs" if i % 2 else "mixed", seed=20 + i)
        for mine, new in zip(d, x):
            mine.copy_(new)
        labels.copy_(torch.randint(0, V, (T,), generator=gen))
        g.copy_(torch.randn(T, generator=gen) * (torch.rand(T, generator=gen) < 0.6))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_a_decoding_step_and_a_training_step(cuda_device):
    """The operators as they are used together: logits of requests with adapters, their tokens with alternatives; then a policy-gradient step
    of the adapters on the log-probabilities."""
    T, H, V, N, R = 96, 256, 4001, 6, 16
    *x, gen = make(T, H, V, N, R, "mixed", seed=12)
    d = on(cuda_device, *x)
    labels = torch.randint(0, V, (T,), generator=gen)
    logits = AD.adapter_logits(*d, dtype=torch.float32)
    r = TU.top_logprobs_from_logits(logits, labels.to(cuda_device), 8, temperature=0.9)
    lsm = torch.log_softmax(plain_logits(*x) / 0.9, 1)
    z_err = float(z_error(*x).max()) / 0.9
    assert float((r.logprobs.cpu().double() - lsm.gather(1, labels[:, None])[:, 0]).abs().max()) <= 2 * z_err + 5e-5
    assert float((r.top_logprobs.cpu().double() - lsm.topk(8, 1).values).abs().max()) <= 2 * z_err + 5e-5
    lp, ent = AD.adapter_logprobs_from_hidden(d[0], d[1], labels.to(cuda_device), d[2].requires_grad_(), d[3].requires_grad_(), d[4], d[5],
                                              temperature=0.9)
    assert float((lp.detach() - r.logprobs).abs().max()) <= 4 * z_err + 1e-4
    advantage = torch.randn(T, generator=gen).to(cuda_device)
    loss = -(torch.exp(lp - r.logprobs) * advantage).mean() - 0.01 * ent.mean()
    loss.backward()
    assert d[2].grad.shape == d[2].shape and bool(torch.isfinite(d[3].grad).all()) and bool(d[3].grad.any())


def test_refusals_of_the_python_entry_points(cuda_device):
    *x, _ = make(8, 64, 100, 2, 8, "mixed")
    d = on(cuda_device, *x)
    y = torch.zeros(8, dtype=torch.int64, device=cuda_device)
    with pytest.raises(TypeError):
        AD.adapter_logits(*d, dtype=torch.float16)
    with pytest.raises(TypeError):
        AD.adapter_logits(d[0].float(), *d[1:])
    with pytest.raises(TypeError):
        AD.adapter_logits(*d[:4], d[4].double(), d[5])
    with pytest.raises(ValueError):
        AD.adapter_logits(*d[:5], d[5][:4])
    with pytest.raises(ValueError):
        AD.adapter_logits(d[0], d[1], d[2][:, :4], d[3][:, :, :4], *d[4:])
    with pytest.raises(ValueError):
        AD.adapter_logits(d[0], d[1], d[2], d[3][:, :50], *d[4:])
    with pytest.raises(ValueError):
        AD.adapter_logits(d[0][:, :60], d[1][:, :60], d[2][:, :, :60], *d[3:])
    with pytest.raises(ValueError):
        AD.adapter_logprobs_from_hidden(d[0], d[1].clone().requires_grad_(), y, *d[2:])
    with pytest.raises(ValueError):
        AD.adapter_logprobs_from_hidden(d[0], d[1], y, *d[2:], temperature=-1.0)
    with pytest.raises(ValueError):
        AD.adapter_logprobs_from_hidden(d[0], d[1], y[:3], *d[2:])
    with pytest.raises(RuntimeError):
        AD.adapter_logits(*x)
    with pytest.raises(ValueError):
        AD.stack_adapters([], [])


@pytest.mark.parametrize("V", [300, 2049])  # d_hidden of a transposed weight, and of one that is read in place
@pytest.mark.parametrize("entropy_grad", [False, True])
def test_the_labels_part_of_the_gradients_is_not_rounded_before_the_result(V, entropy_grad, cuda_device):
    """One token per adapter.  The label's value makes up nearly all of a token's gradients, so its rounding would scale them, by up to e.  The scale
    of a result is its projection on the true one: the roundings of its n elements are independent and at most e each (rms e / sqrt 3), so the
    projection is off by 6 * 0.58 e / sqrt(n) at most, n >= 128, twice that variance where d_hidden is rounded twice (n = 256): 0.31 e.  The other
    columns' roundings add at most e * |p| (the norm of a token's probabilities, below 0.1 for 300 columns): 0.1 e."""
    T, H, R = 40, 256, 128
    *x, gen = make(T, H, V, T, R, seed=V, b_scale=0.02)
    x[1] = (x[1].float() / 4).to(torch.bfloat16)  # logits of about 0.5: p is flat
    x[5] = torch.arange(T)
    labels, g = torch.randperm(V, generator=gen)[:T], torch.randn(T, generator=gen)
    q = 0.1 * torch.randn(T, generator=gen) if entropy_grad else None
    leaves = [t.double().requires_grad_() for t in (x[0], x[2], x[3])]
    z = plain_logits(leaves[0], x[1], leaves[1], leaves[2], x[4], x[5])
    lps = torch.log_softmax(z, dim=1)
    loss = (lps[torch.arange(T), labels] * g.double()).sum()
    if entropy_grad:
        loss = loss - (lps.exp() * lps).sum(1) @ q.double()
    want = torch.autograd.grad(loss, leaves)
    assert float(lps.exp().norm(dim=1).max()) < 0.1
    d, y = on(cuda_device, *x), labels.to(cuda_device)
    _, _, lse, pz = AD.lmhead_adapter_fwd(d[0], d[1], y, *d[2:], 1.0)
    got = AD.lmhead_adapter_bwd(d[0], d[1], y, *d[2:], lse, pz, g.to(cuda_device), None if q is None else q.to(cuda_device), 1.0)
    rows = torch.arange(T)
    for mine, true in zip(got, want):
        mine, true = mine.cpu().double(), true
        if mine.shape[1] == V:  # dB: the label's row
            mine, true = mine[rows, labels], true[rows, labels]
        mine, true = mine.flatten(1), true.flatten(1)
        scale = (mine * true).sum(1) / (true * true).sum(1)
        assert float((scale - 1).abs().max()) <= 0.41 * E, float((scale - 1).abs().max() / E)


def test_last_positions_of_long_sequences_and_dimensions_of_one(cuda_device):
    """Rows further apart than the kernels walk, one row repeated, and strides that mean nothing."""
    *x, gen = make(2, 128, 300, 1, 8, "one", seed=8)
    h, w, a, b, s, ids = on(cuda_device, *x)
    y = torch.randint(0, 300, (2,), generator=gen).to(cuda_device)
    want = AD.adapter_logits(h, w, a, b, s, ids)
    long = torch.zeros((2, 40000, 128), dtype=torch.bfloat16, device=cuda_device)
    long[:, -1] = h
    assert torch.equal(AD.adapter_logits(long[:, -1], w, a, b, s, ids), want)
    assert torch.equal(AD.adapter_logits(long[:1, -1], w, a, b, s, ids[:1]), want[:1])
    odd = lambda t: t.as_strided(t.shape, (3,) + t.stride()[1:])  # noqa: E731  a first dimension of one
    assert torch.equal(AD.adapter_logits(odd(h[:1]), w, odd(a), odd(b), s, ids[:1]), want[:1])
    one = AD.adapter_logits(h, odd(w[:1]), a, b[:, :1].as_strided((1, 1, 8), (8, 3, 1)), s, ids)
    assert float((one.float() - want[:, :1].float()).abs().max()) <= 2 * E * float(want[:, :1].abs().max()) + 1e-3
    row = h[:1].clone().requires_grad_()
    rows = h[:1].expand(2, 128).contiguous().requires_grad_()
    for leaf, use in ((row, lambda: row.expand(2, 128)), (rows, lambda: rows)):
        AD.adapter_logprobs_from_hidden(use(), w, y, a, b, s, ids)[0].sum().backward()
    assert float((row.grad.float() - rows.grad.float().sum(0)).abs().max()) <= E * float(rows.grad.abs().float().sum(0).max())
    with pytest.raises(TypeError):
        AD.adapter_logits(h, w, a, b, s, ids.float())
