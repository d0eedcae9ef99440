"""How far log p(y) is from 64 bits before it is rounded, over many rows: what a
gain over hundreds of tokens adds up.

A margin of one token a sequence, whose reference is that token's 64-bit value
rounded to f32, is the error alone (and the reference's rounding, which is
known): small enough for f32 to hold it.

The exponentials are rounded to f32 one by one; those errors average out over a
row.  What does not is their mean (U / 16 at most is asked for, U = 2^-24: a
mean of one ulp in 32), and the rounding of an f32 sum whose largest term is 1:
+-U there has a root mean square of U / sqrt(3), so U / 4 says that it is not
made."""

import pytest
import torch

from seq_oracle import U
from wap_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k,n", [(112, 2048), (1000, 1024), (5000, 1024), (50001, 512), (140001, 256)])
@pytest.mark.parametrize("peak", [False, True])
def test_errors_do_not_add_up(dtype, k, n, peak):
    r = torch.Generator(device="cuda").manual_seed(k + peak)
    x = torch.randn(n, k, device="cuda", generator=r) * 2
    y = torch.randint(k, (n,), device="cuda", generator=r)
    if peak:  # as of a model that has learned something
        x.scatter_add_(1, y[:, None], torch.randn(n, 1, device="cuda", generator=r) * 2 + 6)
    x = x.to(dtype)
    want = torch.cat([torch.log_softmax(a.double(), -1).gather(-1, b[:, None])[:, 0]
                      for a, b in zip(x.split(64), y.split(64))])
    ref = want.float()
    w = torch.cat([torch.ones(n), torch.zeros(n)]).cuda()
    _, margin = ops.preference_loss(torch.cat([x, x])[:, None], torch.cat([y, y])[:, None],
                                    w[:, None], torch.cat([ref, ref])[:, None], beta=1.0)
    off = margin.double() - (want - ref.double())
    assert off.mean().abs() <= U / 16, float(off.mean() / U)
    assert off.square().mean().sqrt() <= U / 4, float(off.square().mean().sqrt() / U)
