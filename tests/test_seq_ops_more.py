"""Calls of the sequence operators that are allowed and out of the way, on the
CPU's eager form and on the GPU's kernels."""

import math

import pytest
import torch

import seq_oracle as oracle
from seq_oracle import U, assert_within, half_step
from wap_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
pytestmark = pytest.mark.parametrize("device", DEVICES)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def _batch(device, b, t, k, seed, dtype=torch.float32):
    r = gen(seed)
    logits = (torch.randn(b, t, k, generator=r) * 2).to(dtype)
    y = torch.randint(k, (b, t), generator=r)
    w = (torch.rand(b, t, generator=r) < 0.8).float()
    w[0, 0] = 1
    near = torch.log_softmax(logits.double(), -1).gather(-1, y[..., None])[..., 0]
    old, ref = ((near + 0.2 * torch.randn(b, t, generator=r)).float() for _ in range(2))
    adv = torch.randn(b, t, generator=r)
    return [v.to(device) for v in (logits, y, w, old, ref, adv)]


def test_scan_of_one_channel_with_any_upstream_layout(device):
    g = torch.randn(3, 5, 2, generator=gen(0)).to(device).requires_grad_()
    h, last = ops.gated_scan(g)
    up = torch.randn(1, 5, 3, generator=gen(1)).to(device)
    for dh in (up.permute(2, 1, 0), torch.ones(1, device=device).expand(3, 5, 1),
               torch.randn(3, 5, 4, generator=gen(2)).to(device)[..., 1:2]):
        d, = torch.autograd.grad(h, g, dh, retain_graph=True)
        want, bound = oracle.scan(g, None, None, dh, None)["dg"]
        assert_within(d, want, bound + half_step(want, torch.float32))


def test_scan_gates_near_zero_keep_their_relative_precision(device):
    """Small tanh arguments around where its series takes over."""
    n = 512
    size = torch.logspace(-6, 0, n) * torch.where(torch.arange(n) % 2 == 0, 1.0, -1.0)
    g = torch.stack([torch.linspace(-12, 12, n), size], -1)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = g.T.reshape(1, 1, 2 * n).to(dtype).to(device).requires_grad_()
        h, last = ops.gated_scan(x)
        want = oracle.scan(x, None, None, torch.ones(1, 1, n), None)
        v, e = want["last"]
        assert_within(last, v, e + half_step(v, torch.float32))
        d, = torch.autograd.grad(h, x, torch.ones_like(h))
        v, e = want["dg"]
        assert_within(d, v, e + half_step(v, dtype))


def test_scan_nan_gates_are_loud(device):
    for place in (0, 5):
        g = torch.zeros(1, 700, 8, device=device)
        g[0, 300, place] = math.nan
        g.requires_grad_()
        h, last = ops.gated_scan(g)
        c = place % 4
        assert torch.isfinite(h[0, :300]).all() and torch.isnan(h[0, 300:, c]).all()
        assert torch.isnan(last[0, c]) and torch.isfinite(last[0, [i for i in range(4) if i != c]]).all()


def test_scan_states_that_are_not_finite_stay_so(device):
    """Infinity or NaN, the documentation leaves open which: a run of steps is
    one product, and 0.5 ** 200 times infinity is NaN once the product has
    gone under.  Never a finite number, and never another channel's matter."""
    g = torch.zeros(1, 600, 6, device=device)
    for bad in (math.inf, -math.inf, math.nan):
        h0 = torch.tensor([[0.5, bad, 0.5]], device=device)
        h, last = ops.gated_scan(g, h0)
        assert not torch.isfinite(h[0, :, 1]).any() and not torch.isfinite(last[0, 1])
        assert torch.isfinite(h[0, :, [0, 2]]).all() and torch.isfinite(last[0, [0, 2]]).all()


def test_state_in_another_type_and_only_it_wants_a_gradient(device):
    g = torch.randn(2, 300, 6, generator=gen(3)).to(device)
    h0 = torch.randn(2, 3, generator=gen(4)).to(torch.bfloat16).to(device).requires_grad_()
    h, last = ops.gated_scan(g, h0)
    d, = torch.autograd.grad(last.sum(), h0)
    want, bound = oracle.scan(g, h0, None, None, torch.ones(2, 3))["dh0"]
    assert d.dtype == torch.bfloat16
    assert_within(d, want, bound + half_step(want, torch.bfloat16))
    assert not ops.gated_step(g[:, 0], h0)[1].requires_grad


@pytest.mark.parametrize("b,t,k", [(300, 3, 5), (8, 2100, 3)])
def test_preference_of_many_sequences_and_of_many_tokens(device, b, t, k):
    logits, y, w, _, ref, _ = _batch(device, b, t, k, 5)
    logits.requires_grad_()
    want, el, m, em, d, ed = oracle.preference(logits, y, w, ref, 0.2, 0.1)
    loss, margin = ops.preference_loss(logits, y, w, ref, beta=0.2, label_smoothing=0.1)
    assert_within(loss, want, el + 2 * U * want.abs())
    assert_within(margin, m, em + 2 * U * m.abs())
    got, = torch.autograd.grad(loss, logits)
    assert_within(got, d, ed + half_step(d, torch.float32))


def test_no_kl_coefficient_no_kl_term(device):
    """A token that the policy has ruled out lies infinitely far from the
    reference; with kl_coef 0 that is not looked at."""
    logits, y, w, old, ref, adv = _batch(device, 2, 3, 6, 6)
    w = torch.ones_like(w)
    logits[1, 1, y[1, 1]] = -math.inf
    loss, _ = ops.policy_loss(logits, y, w, old, adv, ref, kl_coef=0.0)
    want, _ = ops.policy_loss(logits, y, w, old, adv)
    assert torch.isfinite(loss) and torch.equal(loss, want)
    assert ops.policy_loss(logits, y, w, old, adv, ref, kl_coef=0.1)[0] == math.inf


def test_nan_counts_whatever_its_advantage(device):
    logits, y, w, old, ref, adv = _batch(device, 2, 3, 6, 7)
    w, adv = torch.ones_like(w), torch.zeros_like(adv)
    assert ops.policy_loss(logits, y, w, old, adv)[0] == 0
    bad = logits.clone()
    bad[1, 1, 0] = math.nan
    assert torch.isnan(ops.policy_loss(bad, y, w, old, adv)[0])
    y[0, 0] = 6
    assert torch.isnan(ops.policy_loss(logits, y, w, old, adv)[0])


def test_ratios_that_overflow(device):
    """Clipped where the advantage is positive; infinitely bad where it is
    negative, as the formula says; nothing where it is zero."""
    logits, y, w, old, ref, adv = _batch(device, 1, 3, 6, 8)
    w, old = torch.ones_like(w), torch.full_like(old, -1e4)
    loss, _ = ops.policy_loss(logits, y, w, old, torch.ones_like(adv))
    assert abs(loss.item() + 1.2) < 1e-6
    assert ops.policy_loss(logits, y, w, old, -torch.ones_like(adv))[0] == math.inf
    assert ops.policy_loss(logits, y, w, old, torch.zeros_like(adv))[0] == 0


def test_weights_below_one_and_whole_number_tokens(device):
    logits, y, w, old, ref, adv = _batch(device, 3, 4, 9, 9)
    w = w * 0.05  # the sum stays below one: not divided by
    for yy, ww in ((y, w), (y.int(), w.double()), (y.to(torch.uint8), w)):
        loss, _ = ops.policy_loss(logits, yy, ww, old, adv, ref, kl_coef=0.1)
        want, el, *_ = oracle.policy(logits, y, w, old, adv, ref, 0.2, 0.2, 0.1)
        assert_within(loss, want, el + 2 * U * want.abs())


def test_dropout_with_a_gradient_for_the_residual_alone(device):
    x = torch.randn(4, 9, generator=gen(1)).to(device)
    r = torch.randn(4, 9, generator=gen(2)).to(device).requires_grad_()
    y = ops.counter_dropout(x, 0.5, (1, 2), 0, r)
    dy = torch.randn(9, 4, generator=gen(3)).to(device).t()
    d, = torch.autograd.grad(y, r, dy)
    assert torch.equal(d, dy)
    z = ops.counter_dropout(x.clone().requires_grad_(), 0.5, (1, 2), 0, r.detach())
    assert torch.equal(z, y)


def test_dropout_of_odd_shapes_and_views(device):
    assert ops.counter_dropout(torch.tensor(3.0, device=device), 0.0, (1, 1)) == 3
    x = torch.randn(2, 3, 4, 5, 6, generator=gen(4)).to(device)
    cl = x.to(memory_format=torch.channels_last_3d).requires_grad_()
    y = ops.counter_dropout(cl, 0.5, (2, 2))
    flat = ops.counter_dropout(x.permute(0, 2, 3, 4, 1).contiguous(), 0.5, (2, 2))
    assert torch.equal(y.permute(0, 2, 3, 4, 1), flat)
    d, = torch.autograd.grad(y, cl, torch.ones_like(x))
    assert torch.equal(d != 0, y != 0)
    wide = torch.randn(5, 1, generator=gen(5)).to(device).expand(5, 8)
    assert torch.equal(ops.counter_dropout(wide, 0.5, (3, 3)),
                       ops.counter_dropout(wide.contiguous(), 0.5, (3, 3)))
    counters = torch.tensor([[1, 9], [2, 9]], device=device)
    assert torch.equal(ops.counter_dropout(x, 0.5, counters[:, 0]),
                       ops.counter_dropout(x, 0.5, (1, 2)))


def test_gradients_cannot_be_differentiated_unnoticed(device):
    logits, y, w, old, ref, adv = _batch(device, 2, 3, 6, 10)
    logits.requires_grad_()
    g = torch.randn(2, 3, 4, generator=gen(6)).to(device).requires_grad_()
    x = torch.randn(4, 4, generator=gen(7)).to(device).requires_grad_()
    for out, leaf in ((ops.token_logprob(logits, y, w).sum(), logits),
                      (ops.policy_loss(logits, y, w, old, adv)[0], logits),
                      (ops.preference_loss(logits, y, w, ref)[0], logits),
                      (ops.gated_scan(g)[0].sum(), g),
                      (ops.counter_dropout(x, 0.5, (1, 1)).sum(), x)):
        scale = torch.ones((), device=device, requires_grad=True)
        d, = torch.autograd.grad(out * scale, leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(d.square().sum(), leaf)


def test_inputs_changed_before_the_backward_pass_are_noticed(device):
    logits, y, w, old, ref, adv = _batch(device, 2, 3, 6, 11)
    x = logits.clone().requires_grad_()
    z = x * 1.0
    loss, _ = ops.preference_loss(z, y, w, ref)
    z.mul_(2)
    with pytest.raises(RuntimeError):
        loss.backward()
    g = torch.randn(2, 3, 4, generator=gen(6)).to(device).requires_grad_()
    z = g * 1.0
    h, _ = ops.gated_scan(z)
    z.add_(1)
    with pytest.raises(RuntimeError):
        h.sum().backward()


def test_no_gradient_wanted_none_kept(device):
    logits, y, w, old, ref, adv = _batch(device, 2, 3, 6, 12)
    with torch.no_grad():
        x = logits.clone().requires_grad_()
        assert not ops.policy_loss(x, y, w, old, adv)[0].requires_grad
        assert not ops.token_logprob(x, y).requires_grad
        assert not ops.gated_scan(torch.zeros(1, 2, 4, device=device, requires_grad=True))[0].requires_grad
        assert not ops.counter_dropout(x, 0.5, (1, 1)).requires_grad
