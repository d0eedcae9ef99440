"""The sequence operators have no forward-mode derivative: a tensor that
carries one is refused, it does not come out without it."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from wap_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _calls(device):
    g, h0 = torch.randn(2, 3, 8, device=device), torch.randn(2, 4, device=device)
    x = torch.randn(4, 3, 5, device=device)
    y = torch.zeros(4, 3, dtype=torch.long, device=device)
    w = torch.ones(4, 3, device=device)
    z = torch.randn(6, 7, device=device)
    return {
        "scan": (g, lambda a: ops.gated_scan(a, h0)),
        "scan state": (h0, lambda a: ops.gated_scan(g, a)),
        "logprob": (x, lambda a: ops.token_logprob(a, y, w)),
        "policy": (x, lambda a: ops.policy_loss(a, y, w, w, w, w, kl_coef=0.1)),
        "preference": (x, lambda a: ops.preference_loss(a, y, w, w)),
        "dropout": (z, lambda a: ops.counter_dropout(a, 0.3, (1, 2))),
        "dropout residual": (z, lambda a: ops.counter_dropout(z, 0.3, (1, 2), 0, a)),
    }


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["scan", "scan state", "logprob", "policy",
                                   "preference", "dropout", "dropout residual"])
@pytest.mark.parametrize("tracked", [False, True])
def test_refused(device, which, tracked):
    primal, call = _calls(device)[which]
    with fwd.dual_level():
        dual = fwd.make_dual(primal.clone().requires_grad_(tracked), torch.ones_like(primal))
        with pytest.raises(RuntimeError):
            call(dual)
        with torch.no_grad(), pytest.raises(RuntimeError):
            call(dual)
        # the values alone, as one who wants no derivative asks for them
        call(fwd.unpack_dual(dual).primal.detach())
    call(primal)
