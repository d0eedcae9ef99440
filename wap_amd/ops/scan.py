"""Gated linear recurrence over a sequence: a recurrent cell whose time axis runs in parallel.

::

    z_t = sigmoid(gz_t)      n_t = tanh(gn_t)
    h_t = (1 - z_t) * n_t + z_t * h_{t-1}

The blend is the GRU's (``gru_gates``: packed gates, h' = (1 - z) n + z h)
without the recurrent term inside the gates, so h is linear in the state
before: a whole teacher-forced sequence is one call, its gradient one more,
and decoding is ``gated_step`` once a token.

Dtype policy: gates and h in the caller's dtype (f32, bf16, fp16); the state,
the nonlinearities and every sum in f32 (f64 where the gates are f64, eager
only); h is rounded once.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import op_eager, use_hip
from .functional import _up


def _hip(t: Tensor) -> bool:
    return use_hip(t) and not op_eager("scan")


def _gates(g: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    gz, gn = _up(g).chunk(2, dim=-1)
    return torch.sigmoid(gz), torch.sigmoid(-gz), torch.tanh(gn)


class _GatedScan(torch.autograd.Function):
    """Eager form, step by step (the HIP path has its own node)."""

    @staticmethod
    def forward(ctx, g: Tensor, h0: Optional[Tensor], mask: Optional[Tensor]):
        ctx.set_materialize_grads(False)
        ctx.h0_dtype = None if h0 is None else h0.dtype
        z, zc, n = _gates(g)
        h0 = None if h0 is None else h0.to(n.dtype)
        h = torch.zeros_like(n[:, 0]) if h0 is None else h0
        hs = []
        for t in range(g.shape[1]):
            new = zc[:, t] * n[:, t] + z[:, t] * h
            if mask is not None:
                new = torch.where(mask[:, t, None] > 0, new, h)
            h = new
            hs.append(h)
        ctx.save_for_backward(g, h0, mask)
        return torch.stack(hs, dim=1).to(g.dtype), h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh: Optional[Tensor], dlast: Optional[Tensor]):
        g, h0, mask = ctx.saved_tensors
        if dh is None and dlast is None:
            return None, None, None
        z, zc, n = _gates(g)
        h = torch.zeros_like(n[:, 0]) if h0 is None else h0
        before = []
        for t in range(g.shape[1]):
            before.append(h)
            new = zc[:, t] * n[:, t] + z[:, t] * h
            if mask is not None:
                new = torch.where(mask[:, t, None] > 0, new, h)
            h = new
        c = torch.zeros_like(h) if dlast is None else dlast
        dz, dn = torch.zeros_like(z), torch.zeros_like(n)
        for t in range(g.shape[1] - 1, -1, -1):
            if dh is not None:
                c = c + _up(dh[:, t])
            gz = c * (before[t] - n[:, t]) * z[:, t] * zc[:, t]
            gn = c * zc[:, t] * (1.0 - n[:, t] * n[:, t])
            new = c * z[:, t]
            if mask is not None:
                on = mask[:, t, None] > 0
                gz, gn = torch.where(on, gz, 0.0), torch.where(on, gn, 0.0)
                new = torch.where(on, new, c)
            dz[:, t], dn[:, t], c = gz, gn, new
        dg = torch.cat([dz, dn], dim=-1).to(g.dtype)
        return dg, None if ctx.h0_dtype is None else c.to(ctx.h0_dtype), None


def _check_gates(g: Tensor, dim: int, what: str) -> None:
    if g.dim() != dim or g.shape[-1] % 2:
        raise ValueError(f"{what}: g must be [{'B, T, ' if dim == 3 else 'B, '}"
                         f"2*D], got {tuple(g.shape)}")
    if not g.is_floating_point():
        raise TypeError(f"{what}: g must be floating point, got {g.dtype}")


def _check_state(h: Tensor, g: Tensor, what: str) -> None:
    if tuple(h.shape) != (g.shape[0], g.shape[-1] // 2):
        raise ValueError(f"{what}: state must be [B, D] = "
                         f"{(g.shape[0], g.shape[-1] // 2)}, got {tuple(h.shape)}")
    if h.device != g.device or not h.is_floating_point():
        raise ValueError(f"{what}: state must be floating point on {g.device}")


def gated_scan(g: Tensor, h0: Optional[Tensor] = None,
               mask: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """h[B,T,D] (g's dtype) and the last state[B,D] (f32) of the recurrence
    over packed gates g[B,T,2D] = [z|n], from h0[B,D] (None: zeros).

    mask[B,T] (1 = valid step): a step whose mask is not > 0 leaves the state
    as it is, its gates are not looked at and get a zero gradient; h there is
    the state carried over.  A state that is not finite gives infinities or
    NaN from there on.  Differentiable in g and h0."""
    if g.numel() > 0 and _hip(g):
        from . import ext
        return ext.require().gated_scan(g, h0, mask)
    _check_gates(g, 3, "gated_scan")
    if h0 is not None:
        _check_state(h0, g, "gated_scan")
    if mask is not None:
        if tuple(mask.shape) != tuple(g.shape[:2]) or mask.device != g.device:
            raise ValueError(f"gated_scan: mask must be {tuple(g.shape[:2])} on "
                             f"{g.device}, got {tuple(mask.shape)} on {mask.device}")
        mask = (mask > 0).float() if mask.dtype != torch.float32 else mask
        mask = mask.detach().contiguous()
    if g.numel() == 0:  # nothing to walk over: the state passes through
        b, t, d = g.shape[0], g.shape[1], g.shape[2] // 2
        out = g.reshape(b, t, 2, d)[:, :, 0]
        if h0 is None:
            return out, torch.zeros(b, d, device=g.device, dtype=_up(g).dtype)
        return out, h0.to(_up(g).dtype).clone()
    return _GatedScan.apply(g, h0, mask)


def gated_step(g: Tensor, h: Tensor) -> Tuple[Tensor, Tensor]:
    """One token of :func:`gated_scan` for decoding: (out[B,D] in g's dtype,
    new state[B,D] f32) from gates g[B,2D] and state h[B,D].  Inference only
    (no autograd); ``h`` is not written."""
    if g.numel() > 0 and _hip(g):
        from . import ext
        return ext.require().gated_step(g, h)
    _check_gates(g, 2, "gated_step")
    _check_state(h, g, "gated_step")
    z, zc, n = _gates(g.detach())
    new = zc * n + z * h.detach().to(z.dtype)
    return new.to(g.dtype), new
