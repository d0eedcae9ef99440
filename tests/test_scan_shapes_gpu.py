"""Every cut of the scan's passes against the 64-bit formulas: one and two
channels a lane, each number of waves, chained and not, few and many channel
blocks, and passes that go past the caches."""

import pytest
import torch

from seq_oracle import assert_within, half_step
import seq_oracle as oracle
from wap_amd import ops

pytestmark = pytest.mark.gpu


def _inputs(b, t, d, dtype, seed):
    r = torch.Generator().manual_seed(seed)
    g = torch.randn(b, t, 2 * d, generator=r) * 1.5
    g[..., :d] += 2.0
    m = (torch.rand(b, t, generator=r) < 0.8).float()
    m[-1] = 0
    m[0, t // 2:] = 0  # padded at the end
    if b > 2:
        m[1] = 1
    h0, dl = torch.randn(b, d, generator=r), torch.randn(b, d, generator=r)
    dh = torch.randn(b, t, d, generator=r)
    return [v.cuda() for v in (g.to(dtype), h0, m, dh.to(dtype), dl)]


def _check(g, h0, m, dh, dl):
    g.requires_grad_()
    h0.requires_grad_()
    h, last = ops.gated_scan(g, h0, m)
    dg, dh0 = torch.autograd.grad((h, last), (g, h0), (dh, dl))
    want = oracle.scan(g, h0, m, dh, dl)
    for name, got in (("h", h), ("last", last), ("dg", dg), ("dh0", dh0)):
        v, e = want[name]
        assert_within(got, v, e + half_step(v, got.dtype), name)
    with torch.no_grad():
        again, end = ops.gated_scan(g, h0, m)
    assert torch.equal(again, h) and torch.equal(end, last)


# 64 sequences of 66 channels are 128 channel blocks, half of them nearly
# empty; 67 has one channel a lane
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("t", [1, 8, 9, 12, 16, 17, 30, 33, 60, 64, 65, 100, 128, 129, 200, 256])
@pytest.mark.parametrize("d", [66, 67])
def test_one_tile(t, d, dtype):
    _check(*_inputs(64, t, d, dtype, t + d))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,t,d", [
    (33, 300, 130),   # 99 blocks of 64; two channels a lane: 66
    (64, 257, 66),    # one step in the last tile
    (70, 520, 128),   # more blocks than groups, one each
    (140, 385, 64),   # the same, two a group and not all of them there
    (3, 3000, 1410),  # many tiles behind many blocks
    (4, 1700, 66),    # 8 blocks: one channel a lane
    (65, 400, 63),    # more than 64 blocks of one channel a lane
])
def test_chained(b, t, d, dtype):
    _check(*_inputs(b, t, d, dtype, b + t + d))


@pytest.mark.parametrize("dtype,b,t,d", [
    (torch.bfloat16, 8, 4096, 2048), (torch.float32, 4, 4096, 2048),
    (torch.float16, 70, 700, 1024),
])
def test_past_the_caches(dtype, b, t, d):
    """Gates, h and gradients of more than 256 MB each way; some channels of
    every sequence are compared."""
    r = torch.Generator(device="cuda").manual_seed(b)
    g = torch.randn(b, t, 2 * d, device="cuda", generator=r) * 1.5
    g[..., :d] += 2.0
    g = g.to(dtype).requires_grad_()
    h0 = torch.randn(b, d, device="cuda", generator=r).requires_grad_()
    dh = torch.randn(b, t, d, device="cuda", generator=r).to(dtype)
    dl = torch.randn(b, d, device="cuda", generator=r)
    m = (torch.rand(b, t, device="cuda", generator=r) < 0.9).float()
    m[0, t // 3:] = 0
    assert 3 * b * t * d * g.element_size() > 256 << 20
    h, last = ops.gated_scan(g, h0, m)
    dg, dh0 = torch.autograd.grad((h, last), (g, h0), (dh, dl))
    at = torch.tensor([0, 1, 63, 64, 127, 128, d // 2 - 1, d // 2, d - 65, d - 1], device="cuda")
    gates = torch.cat([at, at + d])
    some = slice(0, b, max(1, b // 4))
    want = oracle.scan(g[some][..., gates], h0[some][:, at], m[some], dh[some][..., at], dl[some][:, at])
    for name, got in (("h", h[some][..., at]), ("last", last[some][:, at]),
                      ("dg", dg[some][..., gates]), ("dh0", dh0[some][:, at])):
        v, e = want[name]
        assert_within(got, v, e + half_step(v, got.dtype), name)
