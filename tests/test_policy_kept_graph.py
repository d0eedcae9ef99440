"""policy_loss: gradients that were handed out are the caller's to write into,
whatever is asked of the same graph afterwards."""

import pytest
import torch

from wap_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _batch(device, b, t, k, seed, dtype=torch.float32):
    r = torch.Generator().manual_seed(seed)
    logits = (torch.randn(b, t, k, generator=r) * 2).to(dtype)
    y = torch.randint(k, (b, t), generator=r)
    w = (torch.rand(b, t, generator=r) < 0.8).float()
    w[0, 0] = 1
    near = torch.log_softmax(logits.double(), -1).gather(-1, y[..., None])[..., 0]
    old, ref = ((near + 0.2 * torch.randn(b, t, generator=r)).float() for _ in range(2))
    adv = torch.randn(b, t, generator=r)
    return [v.to(device) for v in (logits, y, w, old, ref, adv)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("k", [112, 5000, 140001])
def test_written_into_between_two_walks(device, k):
    x, y, w, old, ref, adv = _batch(device, 3, 4, k, 1)
    x.requires_grad_()
    loss, _ = ops.policy_loss(x, y, w, old, adv, ref, kl_coef=0.1)
    first, = torch.autograd.grad(loss, x, retain_graph=True)
    want = first.clone()
    first.mul_(0.5)
    second, = torch.autograd.grad(loss, x, retain_graph=True)
    assert torch.equal(second, want) and torch.equal(first, 0.5 * want)
    second.zero_()
    third, = torch.autograd.grad(loss, x)
    assert torch.equal(third, want)


@pytest.mark.parametrize("device", DEVICES)
def test_accumulated_into_the_same_leaf(device):
    """Clipping or zeroing a leaf's gradient between two passes."""
    x, y, w, old, ref, adv = _batch(device, 2, 3, 60, 2)
    x.requires_grad_()
    loss, _ = ops.policy_loss(x, y, w, old, adv, ref, kl_coef=0.1)
    loss.backward(retain_graph=True)
    want = x.grad.clone()
    x.grad.zero_()
    loss.backward(retain_graph=True)
    assert torch.equal(x.grad, want)
    x.grad.mul_(0.25)
    loss.backward()
    assert torch.equal(x.grad, 1.25 * want)


@pytest.mark.gpu
def test_handed_out_once_and_held_no_longer():
    """A kept graph does not keep the first gradient."""
    x, y, w, old, ref, adv = _batch("cuda", 2, 3, 60, 3)
    x.requires_grad_()
    loss, _ = ops.policy_loss(x, y, w, old, adv, ref)
    d, = torch.autograd.grad(loss, x, retain_graph=True)
    size = torch.cuda.memory_allocated()
    del d
    assert torch.cuda.memory_allocated() < size
    torch.autograd.grad(loss, x)


def _captured(fn, pool, stream):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, pool=pool, stream=stream, capture_error_mode="thread_local"):
        out = fn()
    return g, out


def _drain():
    torch.zeros(1, device="cuda").item()


def _warm(side, x, rest):
    """One pass on the stream that captures, so that nothing is set up there."""
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, w, old, ref, adv = rest
        loss, _ = ops.policy_loss(x, y, w, old, adv, ref, kl_coef=0.1)
        want = torch.autograd.grad(loss, x)[0].clone()
        del loss
    torch.cuda.current_stream().wait_stream(side)
    _drain()
    return want


@pytest.mark.gpu
def test_captured_backward_alone_after_its_result_was_written():
    """Two graphs; the backward one is replayed again after the caller has
    written into the gradient, without the forward one."""
    x, *rest = _batch("cuda", 3, 4, 500, 4)
    y, w, old, ref, adv = rest
    x.requires_grad_()
    up = torch.ones((), device="cuda")
    side, pool = torch.cuda.Stream(), torch.cuda.graph_pool_handle()
    want = _warm(side, x, rest)
    fwd, (loss, _) = _captured(
        lambda: ops.policy_loss(x, y, w, old, adv, ref, kl_coef=0.1), pool, side)
    bwd, (d,) = _captured(lambda: torch.autograd.grad(loss, x, up), pool, side)
    fwd.replay()
    for s in (1.0, 1.0, 2.0, 2.0, 1.0):
        up.fill_(s)
        bwd.replay()
        _drain()
        assert torch.equal(d, s * want), s
        d.mul_(0.5)


@pytest.mark.gpu
def test_forward_captured_and_differentiated_outside():
    """Replays of the forward pass leave gradients alone that were taken from
    its graph outside any capture."""
    x, *rest = _batch("cuda", 3, 4, 500, 5)
    y, w, old, ref, adv = rest
    other = torch.randn(x.shape, generator=torch.Generator().manual_seed(6)).cuda()
    x.requires_grad_()
    side, pool = torch.cuda.Stream(), torch.cuda.graph_pool_handle()
    want = [_warm(side, x, rest)]
    fwd, (loss, _) = _captured(
        lambda: ops.policy_loss(x, y, w, old, adv, ref, kl_coef=0.1), pool, side)
    mine = x.detach().clone()
    x.data.copy_(other)
    want.append(_warm(side, other.clone().requires_grad_(), rest))
    got = []
    for v in (mine, other):
        x.data.copy_(v)
        fwd.replay()
        _drain()
        got.append(torch.autograd.grad(loss, x, retain_graph=True)[0])
        _drain()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i]), i
