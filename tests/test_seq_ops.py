"""Sequence operators on the CPU: the eager path against the 64-bit formulas
and finite differences, and what the entry points refuse."""

import math

import pytest
import torch

import seq_oracle as oracle
from wap_amd import ops
from wap_amd.ops import seqloss
from wap_amd.ops.scan import _GatedScan

F64 = torch.float64


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------ gated recurrence

@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("start", [False, True])
@pytest.mark.parametrize("b,t,d", [(1, 1, 1), (3, 7, 5), (2, 20, 9)])
def test_scan_is_the_formula(b, t, d, mask, start):
    r = gen(b * 100 + t)
    g = torch.randn(b, t, 2 * d, generator=r, dtype=F64).requires_grad_()
    h0 = torch.randn(b, d, generator=r, dtype=F64).requires_grad_() if start else None
    m = (torch.rand(b, t, generator=r) < 0.6).float() if mask else None
    if mask and b > 1:
        m[1] = 0
    dh = torch.randn(b, t, d, generator=r, dtype=F64)
    dl = torch.randn(b, d, generator=r, dtype=F64)
    h, last = ops.gated_scan(g, h0, m)
    want = oracle.scan(g, h0, m, dh, dl)
    torch.testing.assert_close(h, want["h"][0])
    torch.testing.assert_close(last, want["last"][0])
    grads = torch.autograd.grad((h, last), (g, h0) if start else (g,), (dh, dl))
    torch.testing.assert_close(grads[0], want["dg"][0])
    if start:
        torch.testing.assert_close(grads[1], want["dh0"][0])


def test_scan_gradcheck():
    r = gen(5)
    g = torch.randn(2, 6, 6, generator=r, dtype=F64).requires_grad_()
    h0 = torch.randn(2, 3, generator=r, dtype=F64).requires_grad_()
    m = torch.ones(2, 6)
    m[0, 2] = m[1, 4:] = 0
    for mask in (None, m):
        assert torch.autograd.gradcheck(lambda a, b: ops.gated_scan(a, b, mask), (g, h0))
    assert torch.autograd.gradcheck(lambda a: ops.gated_scan(a)[1], (g,))


def test_scan_step_by_step_is_the_whole():
    r = gen(6)
    g, h = torch.randn(3, 9, 8, generator=r), torch.randn(3, 4, generator=r)
    want, last = ops.gated_scan(g, h)
    for t in range(9):
        out, h = ops.gated_step(g[:, t], h)
        torch.testing.assert_close(out, want[:, t])
    torch.testing.assert_close(h, last)


def test_scan_masked_gates_are_not_looked_at():
    g = torch.randn(2, 5, 6, generator=gen(7))
    m = torch.ones(2, 5)
    m[0, 3:] = m[1, :] = 0
    clean = g.clone()
    g[m == 0] = math.nan
    g.requires_grad_()
    h, last = ops.gated_scan(g, None, m)
    torch.testing.assert_close(h, ops.gated_scan(clean, None, m)[0])
    assert (h[1] == 0).all() and (last[1] == 0).all()
    (dg,) = torch.autograd.grad(h.sum(), g)
    assert (dg[m == 0] == 0).all() and torch.isfinite(dg).all()


@pytest.mark.parametrize("b,t,d", [(0, 3, 4), (2, 0, 4), (2, 3, 0)])
def test_scan_of_nothing(b, t, d):
    g = torch.randn(b, t, 2 * d).requires_grad_()
    h0 = torch.randn(b, d).requires_grad_()
    h, last = ops.gated_scan(g, h0)
    assert h.shape == (b, t, d) and torch.equal(last, h0)
    dg, dh0 = torch.autograd.grad(h.sum() + last.sum(), (g, h0))
    assert dg.shape == g.shape and torch.equal(dh0, torch.ones_like(h0))
    assert ops.gated_scan(g)[1].shape == (b, d)


def test_scan_refusals():
    g = torch.randn(2, 3, 8)
    for bad in (torch.randn(2, 3, 7), torch.randn(2, 8)):
        with pytest.raises(ValueError):
            ops.gated_scan(bad)
    with pytest.raises(TypeError):
        ops.gated_scan(torch.ones(2, 3, 8, dtype=torch.long))
    with pytest.raises(ValueError):
        ops.gated_scan(g, torch.zeros(2, 8))
    with pytest.raises(ValueError):
        ops.gated_scan(g, None, torch.ones(3, 2))
    with pytest.raises(ValueError):
        ops.gated_step(g, torch.zeros(2, 4))
    with pytest.raises(ValueError):
        ops.gated_step(g[:, 0], torch.zeros(2, 3))


# ------------------------------------------------------ token probabilities

def _batch(b, t, k, seed=0, dtype=F64):
    r = gen(seed)
    logits = torch.randn(b, t, k, generator=r, dtype=dtype) * 2
    y = torch.randint(k, (b, t), generator=r)
    w = (torch.rand(b, t, generator=r) < 0.7).float()
    w[-1] = 0
    near = torch.log_softmax(logits, -1).gather(-1, y[..., None])[..., 0]
    old = near + 0.3 * torch.randn(b, t, generator=r, dtype=dtype)
    ref = near + 0.2 * torch.randn(b, t, generator=r, dtype=dtype)
    adv = torch.randn(b, t, generator=r, dtype=dtype)
    return logits.requires_grad_(), y, w, old, ref, adv


@pytest.mark.parametrize("b,t,k", [(1, 1, 1), (2, 3, 5), (4, 6, 112)])
def test_token_logprob_is_log_softmax(b, t, k):
    logits, y, w, *_ = _batch(b, t, k)
    got = ops.token_logprob(logits, y)
    want = torch.log_softmax(logits, -1).gather(-1, y[..., None])[..., 0]
    torch.testing.assert_close(got, want)
    up = torch.randn(b, t, dtype=F64)
    a, = torch.autograd.grad(got, logits, up)
    c, = torch.autograd.grad(want, logits, up)
    torch.testing.assert_close(a, c)
    masked = ops.token_logprob(logits, y, w)
    torch.testing.assert_close(masked, want * w)


@pytest.mark.parametrize("kl,with_ref", [(0.0, False), (0.1, True)])
@pytest.mark.parametrize("per_seq", [False, True])
def test_policy_loss_is_its_formula(kl, with_ref, per_seq):
    logits, y, w, old, ref, adv = _batch(4, 6, 11, seed=3)
    adv = adv[:, 0] if per_seq else adv
    loss, logp = ops.policy_loss(logits, y, w, old, adv, ref if with_ref else None,
                                 clip_low=0.2, clip_high=0.3, kl_coef=kl)
    lp = torch.log_softmax(logits, -1).gather(-1, y[..., None])[..., 0]
    a = adv[:, None] if per_seq else adv
    ratio = torch.exp(lp - old)
    l = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.3) * a)
    l = l + kl * (torch.exp(ref - lp) - (ref - lp) - 1)
    want = (l * w).sum() / w.sum()
    torch.testing.assert_close(loss, want)
    torch.testing.assert_close(logp, (lp * w).detach())
    assert not logp.requires_grad
    torch.testing.assert_close(torch.autograd.grad(loss, logits)[0],
                               torch.autograd.grad(want, logits)[0])


def test_losses_gradcheck():
    logits, y, w, old, ref, adv = _batch(4, 3, 5, seed=11)
    w = w * torch.tensor([[0.5], [1.0], [2.0], [1.0]])
    assert torch.autograd.gradcheck(lambda x: ops.token_logprob(x, y, w), (logits,))
    assert torch.autograd.gradcheck(
        lambda x: ops.policy_loss(x, y, w, old, adv, ref, kl_coef=0.2)[0], (logits,))
    for s in (0.0, 0.1):
        assert torch.autograd.gradcheck(
            lambda x: ops.preference_loss(x, y, w, ref, beta=0.7, label_smoothing=s)[0],
            (logits,))


@pytest.mark.parametrize("eps", [0.0, 0.25])
def test_preference_loss_is_its_formula(eps):
    logits, y, w, _, ref, _ = _batch(6, 5, 13, seed=4)
    loss, margin = ops.preference_loss(logits, y, w, ref, beta=0.5, label_smoothing=eps)
    lp = torch.log_softmax(logits, -1).gather(-1, y[..., None])[..., 0]
    gain = ((lp - ref) * w).sum(1)
    m = 0.5 * (gain[:3] - gain[3:])
    ls = torch.nn.functional.logsigmoid
    want = -((1 - eps) * ls(m) + eps * ls(-m)).mean()
    torch.testing.assert_close(loss, want)
    torch.testing.assert_close(margin, m.detach())
    torch.testing.assert_close(torch.autograd.grad(loss, logits)[0],
                               torch.autograd.grad(want, logits)[0])


def test_policy_at_a_border_the_unclipped_side_counts():
    one = torch.tensor([0.0, 0.0], dtype=F64)
    adv = torch.tensor([2.0, -2.0], dtype=F64)
    loss, slope = seqloss._policy_terms(one, one, adv, None, 0.0, 0.0, 0.0)
    assert torch.equal(loss, -adv) and torch.equal(slope, -adv)
    # one of the two sides further on: clipped where the advantage favours it
    loss, slope = seqloss._policy_terms(one + 0.1, one, adv, None, 0.0, 0.0, 0.0)
    assert loss[0] == -2 and slope[0] == 0 and slope[1] == 2 * math.exp(0.1)


def test_policy_zero_advantage_of_a_ratio_that_overflows():
    far = torch.tensor([1e4], dtype=F64)
    loss, slope = seqloss._policy_terms(far, far * 0, far * 0, None, 0.2, 0.2, 0.0)
    assert loss.item() == 0 and slope.item() == 0


def test_masked_rows_may_hold_anything():
    logits, y, w, old, ref, adv = _batch(4, 6, 9, seed=8, dtype=torch.float32)
    clean = [v.detach().clone() for v in (logits, old, ref, adv)]
    off = w == 0
    with torch.no_grad():
        logits[off] = math.nan
    for v in (old, ref, adv):
        v[off] = math.inf
    y = torch.where(off, -100, y)
    for x, (o, r, a), yy in ((logits, (old, ref, adv), y),
                             (clean[0].requires_grad_(), clean[1:], y.clamp_min(0))):
        l1, lp = ops.policy_loss(x, yy, w, o, a, r, kl_coef=0.1)
        l2, _ = ops.preference_loss(x, yy, w, r)
        grads = [torch.autograd.grad(l, x)[0] for l in (l1, l2)]
        assert all((d[off] == 0).all() for d in grads)
        now = (l1.detach(), l2.detach(), lp, *grads)
        if x is logits:
            first = now
    for u, v in zip(first, now):
        assert torch.equal(u, v)


def test_nothing_counts():
    logits, y, w, old, ref, adv = _batch(2, 3, 4)
    w = torch.zeros_like(w)
    loss, _ = ops.policy_loss(logits, y, w, old, adv, ref, kl_coef=1.0)
    assert loss.item() == 0
    assert (torch.autograd.grad(loss, logits)[0] == 0).all()
    loss, margin = ops.preference_loss(logits, y, w, ref)
    assert margin.item() == 0 and abs(loss.item() - math.log(2)) < 1e-12
    assert (torch.autograd.grad(loss, logits)[0] == 0).all()


def test_tokens_outside_the_vocabulary_are_loud():
    logits, y, w, old, ref, adv = _batch(2, 3, 4)
    w = torch.ones_like(w)
    for bad in (-1, 4):
        y[1, 2] = bad
        assert torch.isnan(ops.token_logprob(logits, y))[1, 2]
        assert torch.isnan(ops.policy_loss(logits, y, w, old, adv)[0])
        assert torch.isnan(ops.preference_loss(logits, y, w, ref)[0])


def test_backward_twice_and_scaled():
    logits, y, w, old, ref, adv = _batch(4, 3, 7, seed=2)
    loss, _ = ops.policy_loss(logits, y, w, old, adv, ref, kl_coef=0.1)
    a, = torch.autograd.grad(loss, logits, retain_graph=True)
    b, = torch.autograd.grad(loss, logits, torch.tensor(3.0, dtype=F64))
    torch.testing.assert_close(3 * a, b)


def test_loss_refusals():
    logits, y, w, old, ref, adv = _batch(2, 3, 4)
    with pytest.raises(ValueError):
        ops.token_logprob(logits[0], y[0])
    with pytest.raises(ValueError):
        ops.token_logprob(logits, y[:, :2])
    with pytest.raises(TypeError):
        ops.token_logprob(logits, y.double())
    with pytest.raises(TypeError):
        ops.token_logprob(logits.detach().long(), y)
    with pytest.raises(ValueError):
        ops.token_logprob(logits, y, w[:1])
    with pytest.raises(ValueError):
        ops.policy_loss(logits, y, None, old, adv)
    with pytest.raises(ValueError):
        ops.policy_loss(logits, y, w, old[:, :1], adv)
    with pytest.raises(ValueError):
        ops.policy_loss(logits, y, w, old, adv[:, :2])
    with pytest.raises(ValueError):
        ops.policy_loss(logits, y, w, old, adv, clip_low=-0.1)
    with pytest.raises(ValueError):
        ops.policy_loss(logits[:0], y[:0], w[:0], old[:0], adv[:0])
    with pytest.raises(ValueError):
        ops.preference_loss(logits[:1], y[:1], w[:1], ref[:1])
    with pytest.raises(ValueError):
        ops.preference_loss(logits, y, w, None)
    with pytest.raises(ValueError):
        ops.preference_loss(logits, y, w, ref, label_smoothing=1.5)


# ------------------------------------------------------ dropout

def test_generator_has_the_published_values():
    """Known answers of Philox4x32 with seven rounds, as its authors publish
    them with their generator: all bits zero, all bits one."""
    u = oracle.draws(8, 0, 0, 0)
    words = [int(u[2 * i]) | int(u[2 * i + 1]) << 16 for i in range(4)]
    assert words == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]


@pytest.mark.parametrize("seed,step,stream", [(0, 0, 0), (-3, 7, 1), (2 ** 40 + 5, 2 ** 35, 2 ** 24 - 1)])
@pytest.mark.parametrize("n", [1, 8, 37])
def test_dropout_mask_is_the_generators(n, seed, step, stream):
    x = torch.randn(n, generator=gen(n)) + 5.0
    want, bound, keep = oracle.dropout(x, 0.4, seed, step, stream)
    y = ops.counter_dropout(x, 0.4, (seed, step), stream)
    assert torch.equal(y != 0, keep)
    oracle.assert_within(y, want, bound)
    at = torch.tensor([seed, step])
    assert torch.equal(ops.counter_dropout(x, 0.4, at, stream), y)


def test_dropout_backward_uses_the_forwards_draws():
    x = torch.randn(5, 11, generator=gen(1)).requires_grad_()
    res = torch.randn(5, 11, generator=gen(2)).requires_grad_()
    rng = torch.tensor([3, 0])
    y = ops.counter_dropout(x, 0.3, rng, 2, res)
    rng[1] += 1
    dy = torch.randn(5, 11, generator=gen(3))
    dx, dres = torch.autograd.grad(y, (x, res), dy)
    want, bound, keep = oracle.dropout(dy, 0.3, 3, 0, 2)
    assert torch.equal(dx != 0, keep)
    oracle.assert_within(dx, want, bound)
    assert torch.equal(dres, dy)
    z = ops.counter_dropout(x, 0.3, rng, 2, res)
    assert not torch.equal(y, z)


def test_dropout_shares_mean_and_ends():
    x = torch.full((200_000,), 1.0)
    y = ops.counter_dropout(x, 0.3, (1, 2))
    share = (y == 0).float().mean().item()
    # five standard deviations of 200000 draws
    assert abs(share - 0.3) < 5 * math.sqrt(0.3 * 0.7 / 200_000)
    assert torch.equal(ops.counter_dropout(x, 0.0, (1, 2)), x)
    assert (ops.counter_dropout(x, 1.0, (1, 2)) == 0).all()
    assert not torch.equal(y, ops.counter_dropout(x, 0.3, (1, 2), stream=1))
    assert not torch.equal(y, ops.counter_dropout(x, 0.3, (1, 3)))
    assert not torch.equal(y, ops.counter_dropout(x, 0.3, (2, 2)))


def test_dropout_drops_nan_and_follows_memory_order():
    x = torch.full((64,), math.nan)
    y = ops.counter_dropout(x, 0.5, (0, 0))
    keep = oracle.dropout(torch.ones(64), 0.5, 0, 0, 0)[2]
    assert torch.equal(torch.isnan(y), keep) and (y[~keep] == 0).all()
    x = torch.randn(2, 3, 4, 5, generator=gen(9)).to(memory_format=torch.channels_last)
    x.requires_grad_()
    y = ops.counter_dropout(x, 0.5, (4, 4))
    flat = x.detach().permute(0, 2, 3, 1).contiguous()
    assert y.is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(y.permute(0, 2, 3, 1), ops.counter_dropout(flat, 0.5, (4, 4)))
    # an upstream gradient in another order meets the same mask
    dx, = torch.autograd.grad(y, x, torch.ones(2, 3, 4, 5))
    assert torch.equal(dx != 0, y != 0)


def test_dropout_gradcheck():
    x = torch.randn(3, 5, dtype=F64, generator=gen(3)).requires_grad_()
    r = torch.randn(3, 5, dtype=F64, generator=gen(4)).requires_grad_()
    assert torch.autograd.gradcheck(
        lambda a, b: ops.counter_dropout(a, 0.4, (1, 1), 0, b), (x, r))


def test_dropout_refusals():
    x = torch.randn(4, 4)
    for p in (-0.1, 1.1, math.nan):
        with pytest.raises(ValueError):
            ops.counter_dropout(x, p, (0, 0))
    with pytest.raises(ValueError):
        ops.counter_dropout(x, 0.1, (0, 0), stream=1 << 24)
    with pytest.raises(ValueError):
        ops.counter_dropout(x, 0.1, (0,))
    with pytest.raises(ValueError):
        ops.counter_dropout(x, 0.1, torch.zeros(2))
    with pytest.raises(ValueError):
        ops.counter_dropout(x, 0.1, (0, 0), residual=torch.randn(4, 5))
    with pytest.raises(ValueError):
        ops.counter_dropout(x, 0.1, (0, 0), residual=torch.randn(4, 4).half())
    with pytest.raises(TypeError):
        ops.counter_dropout(x.long(), 0.1, (0, 0))


# ------------------------------------------------------ together

def _layer(p, x, h0, mask, rng):
    """A decoder layer as the operators are used together."""
    emb = p["emb"][x]
    h, last = ops.gated_scan(emb @ p["w"], h0, mask)
    h = ops.counter_dropout(h, 0.2, rng, stream=1, residual=emb)
    return h @ p["o"], last


def test_together_gradients_against_differences():
    r = gen(21)
    p = {n: (torch.randn(*s, generator=r, dtype=F64) * 0.5).requires_grad_()
         for n, s in (("emb", (7, 4)), ("w", (4, 8)), ("o", (4, 7)))}
    x = torch.randint(7, (4, 5), generator=r)
    y = torch.randint(7, (4, 5), generator=r)
    mask = torch.ones(4, 5)
    mask[1, 3:] = mask[2, 1:] = 0
    with torch.no_grad():
        logits, _ = _layer(p, x, None, mask, (1, 0))
        old = ops.token_logprob(logits, y, mask) + 0.1
    adv = torch.randn(4, generator=r, dtype=F64)

    def loss(emb, w, o):
        logits, last = _layer(dict(emb=emb, w=w, o=o), x, None, mask, (1, 0))
        a, _ = ops.policy_loss(logits, y, mask, old, adv, old, kl_coef=0.1)
        b, _ = ops.preference_loss(logits, y, mask, old, beta=0.5)
        return a + b + last.square().sum()

    assert torch.autograd.gradcheck(loss, tuple(p.values()))


def test_scan_function_is_once_differentiable():
    g = torch.randn(1, 3, 4, dtype=F64, requires_grad=True)
    h, _ = _GatedScan.apply(g, None, None)
    d, = torch.autograd.grad(h.sum(), g, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), g)
