"""Gates far out, where z = sigmoid(gz) nears the smallest f32 numbers: it
keeps its relative precision down to there."""

import pytest
import torch

from seq_oracle import U, assert_within
from wap_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t", [1, 300])
def test_forgotten_state_is_what_the_gate_leaves(device, dtype, t):
    """n = 0: h = z h0 and dgz = h0 z (1 - z), both of the size of z."""
    gz = torch.linspace(-87.0, -70.0, 137).to(dtype)
    d = gz.numel()
    g = torch.zeros(1, t, 2 * d, dtype=dtype)
    g[0, 0, :d] = gz
    g[0, 1:, :d] = 200.0  # z = 1: kept from there on
    h0 = torch.ones(1, d)
    x = g.to(device).requires_grad_()
    h, last = ops.gated_scan(x, h0.to(device))
    want = torch.sigmoid(gz.double())[None]
    # e = 2^u with u = -gz log2 e: u's rounding and that of log2 e, u U each,
    # times ln 2, the exponential's and the reciprocal's 2 ulp each
    size = (2 * 126 * 0.7 + 8) * U
    assert_within(last, want, size * want, "last")
    dlast = torch.ones_like(last)
    dg, = torch.autograd.grad(last, x, dlast)
    if dtype != torch.float16:  # whose smallest number is far above
        got = dg[:, 0, :d]
        step = torch.finfo(dtype).eps / 2
        assert_within(got, want * (1 - want), (size + 8 * U + step) * want, "dgz")
    out, new = ops.gated_step(x[:, 0].detach(), h0.to(device))
    assert_within(new, want, size * want, "step")
