"""preference_loss where a sequence holds a token that the policy has ruled
out (probability zero): one margin is infinite, the loss of that pair is what
-log sigmoid of it is, and the other pairs keep theirs."""

import math

import pytest
import torch

import seq_oracle as oracle
from seq_oracle import U, assert_within, half_step
from wap_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _softplus(m):
    return torch.logaddexp(torch.zeros_like(m), m)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("pairs,t", [(2, 3), (150, 3), (3, 2100)])
@pytest.mark.parametrize("eps", [0.0, 0.1, 1.0])
@pytest.mark.parametrize("which", ["rejected", "preferred"])
def test_infinite_margin(device, pairs, t, eps, which):
    k, beta = 5, 0.3
    r = torch.Generator().manual_seed(pairs + t)
    logits = torch.randn(2 * pairs, t, k, generator=r) * 2
    y = torch.randint(k, (2 * pairs, t), generator=r)
    w = torch.ones(2 * pairs, t)
    ref = torch.log_softmax(logits.double(), -1).gather(-1, y[..., None])[..., 0]
    ref = (ref + 0.2 * torch.randn(2 * pairs, t, generator=r)).float()
    seq = 2 * pairs - 1 if which == "rejected" else pairs - 1  # of the last pair
    logits[seq, 1, y[seq, 1]] = -math.inf

    logp, elog, p, ep, at, live = oracle.rows(logits, y, w)
    gain = (logp - ref.double()).sum(1)
    m = beta * (gain[:pairs] - gain[pairs:])
    em = beta * (elog.sum(1)[:pairs] + elog.sum(1)[pairs:])
    assert m[-1] == (math.inf if which == "rejected" else -math.inf)
    assert torch.isfinite(m[:-1]).all()
    # a term of coefficient zero is no term, as in the limit of the margin
    each = torch.zeros_like(m)
    if eps < 1:
        each = each + (1 - eps) * _softplus(-m)
    if eps > 0:
        each = each + eps * _softplus(m)
    want = each.mean()
    finite = (which, eps) in (("rejected", 0.0), ("preferred", 1.0))
    assert bool(torch.isfinite(want)) == finite

    x = logits.to(device).requires_grad_()
    loss, margin = ops.preference_loss(x, y.to(device), w.to(device), ref.to(device),
                                       beta=beta, label_smoothing=eps)
    assert_within(loss, want, em.mean() + 2 * U * want.abs(), "loss")
    assert_within(margin, m, em + 2 * U * m.abs(), "margin")
    got, = torch.autograd.grad(loss, x)
    *_, d, ed = oracle.preference(logits, y, w, ref, beta, eps)
    assert_within(got, d, ed + half_step(d, torch.float32), "dlogits")
    assert torch.isfinite(got).all()
