"""token_logprob of a token outside the vocabulary: NaN, and where anything
depends on it so is its row's gradient; the other rows keep theirs."""

import pytest
import torch

import seq_oracle as oracle
from seq_oracle import DTYPES, assert_within, half_step
from wap_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [1, 6, 300, 5000])
@pytest.mark.parametrize("bad", [-1, None, 1 << 40, -(1 << 40)])
def test_gradient(device, dtype, k, bad):
    r = torch.Generator().manual_seed(k)
    logits = (torch.randn(3, 4, k, generator=r) * 2).to(dtype)
    y = torch.randint(k, (3, 4), generator=r)
    up = torch.randn(3, 4, generator=r)
    w = torch.ones(3, 4)
    w[2, 1] = 0
    bad = k if bad is None else bad
    y[0, 1] = y[1, 3] = y[2, 1] = bad
    up[1, 3] = 0  # as where the NaN was replaced downstream
    x = logits.to(device).requires_grad_()
    logp = ops.token_logprob(x, y.to(device), w.to(device))
    assert torch.isnan(logp[0, 1]) and torch.isnan(logp[1, 3]) and logp[2, 1] == 0
    d, = torch.autograd.grad(logp, x, up.to(device))
    d = d.cpu()
    assert torch.isnan(d[0, 1]).all()
    assert (d[1, 3] == 0).all() and (d[2, 1] == 0).all()
    good = torch.ones(3, 4, dtype=torch.bool)
    good[0, 1] = good[1, 3] = good[2, 1] = False
    _, _, p, ep, at, live = oracle.rows(logits, y, w)
    want, bound = oracle.rows_grad(up.double(), torch.zeros(3, 4, dtype=torch.float64), p, ep, at, live)
    assert_within(d[good], want[good], (bound + half_step(want, dtype))[good])


@pytest.mark.parametrize("device", DEVICES)
def test_losses(device):
    r = torch.Generator().manual_seed(1)
    x = torch.randn(4, 3, 7, generator=r).to(device).requires_grad_()
    y = torch.randint(7, (4, 3), generator=r).to(device)
    w = torch.ones(4, 3, device=device)
    y[1, 2] = 7
    loss, _ = ops.policy_loss(x, y, w, w, 0 * w)
    d, = torch.autograd.grad(loss, x)
    assert torch.isnan(loss) and torch.isnan(d[1, 2]).all()
    d[1, 2] = 0
    assert torch.isfinite(d).all()
    loss, _ = ops.preference_loss(x, y, w, w)
    d, = torch.autograd.grad(loss, x)
    # the pair's margin is NaN, and every token of the pair depends on it
    assert torch.isnan(loss) and torch.isnan(d[1]).all() and torch.isnan(d[3]).all()
    assert torch.isfinite(d[0]).all() and torch.isfinite(d[2]).all()
