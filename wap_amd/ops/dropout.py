"""Dropout from a counter-based generator: the mask is a function of (seed,
step, stream, place) and is never stored.

The generator is Philox4x32 of Salmon, Moraes, Dror and Shaw ("Parallel random
numbers: as easy as 1, 2, 3", SC 2011) with seven rounds; a call of it gives
eight 16-bit draws, for eight elements next to each other in memory.  An
element is kept where its draw is >= limit = round(p * 2**16) and scaled by
2**16 / (2**16 - limit), the inverse of the share that is really kept.

The backward pass makes the draws again.  With (seed, step) in a device tensor
that the program advances, a captured step drops other elements at every
replay.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence, Union

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import op_eager, use_hip
from .functional import _up

_LOW = 0xFFFFFFFF


def _hip(t: Tensor) -> bool:
    return use_hip(t) and not op_eager("dropout")


def _limit(p: float) -> int:
    return math.floor(p * 65536 + 0.5)


def _words(c0: Tensor, c1: Tensor, c2: Tensor, c3: Tensor, k0: Tensor,
           k1: Tensor) -> Tensor:
    """The generator's four words [..., 4] of a counter and a key (32 bits
    each, in int64 arithmetic, wrapping)."""
    for _ in range(7):
        p, q = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((q >> 32) & _LOW) ^ c1 ^ k0, q & _LOW,
                          ((p >> 32) & _LOW) ^ c3 ^ k1, p & _LOW)
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return torch.stack([c0, c1, c2, c3], dim=-1)


def _draws(n: int, rng: Tensor, stream: int) -> Tensor:
    """The n 16-bit draws in storage order."""
    group = torch.arange((n + 7) // 8, device=rng.device)
    c0, c1 = group & _LOW, (stream << 8) | (group >> 32)
    c2 = (rng[1] & _LOW).expand_as(c0)
    c3 = ((rng[1] >> 32) & _LOW).expand_as(c0)
    words = _words(c0, c1, c2, c3, rng[0] & _LOW, (rng[0] >> 32) & _LOW)
    return torch.stack([words & 0xFFFF, words >> 16], dim=-1).view(-1)[:n]


def _apply(x: Tensor, residual: Optional[Tensor], p: float, rng: Tensor,
           stream: int) -> Tensor:
    """Of a contiguous x (eager; the HIP path has its own node)."""
    limit = _limit(p)
    on = (_draws(x.numel(), rng, stream) >= limit).view(x.shape)
    scale = 65536 / (65536 - limit) if limit < 65536 else 0.0
    y = torch.where(on, _up(x) * scale, 0.0)
    if residual is not None:
        y = y + _up(residual)
    return y.to(x.dtype)


def _in_order(t: Tensor, fmt: Optional[torch.memory_format]) -> Tensor:
    """`t` as a contiguous tensor whose order is the storage order of `fmt`."""
    if fmt is None:
        return t.contiguous()
    dims = (0, *range(2, t.dim()), 1)
    return t.contiguous(memory_format=fmt).permute(dims)


def _back(t: Tensor, fmt: Optional[torch.memory_format]) -> Tensor:
    if fmt is None:
        return t
    return t.permute(0, t.dim() - 1, *range(1, t.dim() - 1))


class _CounterDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, residual: Optional[Tensor], p: float, rng,
                stream: int):
        fmt = None
        if not x.is_contiguous():
            last = {4: torch.channels_last, 5: torch.channels_last_3d}.get(x.dim())
            if last is not None and x.is_contiguous(memory_format=last):
                fmt = last
        rng = (rng.clone() if isinstance(rng, Tensor)
               else torch.tensor(rng, dtype=torch.int64, device=x.device))
        y = _apply(_in_order(x, fmt),
                   None if residual is None else _in_order(residual, fmt),
                   p, rng, stream)
        ctx.meta = (p, stream, fmt, residual is not None)
        ctx.save_for_backward(rng)
        return _back(y, fmt)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy: Tensor):
        p, stream, fmt, has_res = ctx.meta
        dx = None
        if ctx.needs_input_grad[0]:
            rng, = ctx.saved_tensors
            dx = _back(_apply(_in_order(dy, fmt), None, p, rng, stream), fmt)
        dres = dy if has_res and ctx.needs_input_grad[1] else None
        return dx, dres, None, None, None


def _signed(v: int) -> int:
    """A 64-bit pattern as the int64 that holds it."""
    v &= (1 << 64) - 1
    return v - (1 << 64) if v >> 63 else v


def counter_dropout(x: Tensor, p: float, rng: Union[Tensor, Sequence[int]],
                    stream: int = 0,
                    residual: Optional[Tensor] = None) -> Tensor:
    """x with a share p of its elements zeroed and the others scaled, plus
    ``residual`` (one rounding of the sum).

    ``rng``: (seed, step) as two integers, or an int64 tensor [2] on x's
    device, read when the kernel runs; the backward pass uses the pair that
    the forward pass read, also if the tensor has been advanced since.
    ``stream`` (0 <= stream < 2**24) keeps layers of one step apart.

    The mask follows x's order in memory: a contiguous x, or one in
    channels-last order; anything else is made contiguous first.  A dropped
    NaN or infinity is dropped.  Differentiable in x and residual."""
    if not x.is_floating_point():
        raise TypeError(f"counter_dropout: x must be floating point, got {x.dtype}")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"counter_dropout: p must be in [0, 1], got {p}")
    if not 0 <= stream < 1 << 24:
        raise ValueError(f"counter_dropout: stream must be in [0, 2**24), got {stream}")
    at = None
    if isinstance(rng, Tensor):
        at = rng
    elif len(rng) == 2:
        rng = (_signed(int(rng[0])), _signed(int(rng[1])))
    else:
        raise ValueError("counter_dropout: rng must be (seed, step)")
    if _hip(x):
        from . import ext
        seed, step = (0, 0) if at is not None else rng
        return ext.require().counter_dropout(x, residual, p, at, seed, step, stream)
    if at is not None and (at.dtype != torch.int64 or tuple(at.shape) != (2,)
                           or at.device != x.device):
        raise ValueError("counter_dropout: rng must be int64 [2] on "
                         f"{x.device}, got {at.dtype} {tuple(at.shape)} on {at.device}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype
                                 or residual.device != x.device):
        raise ValueError("counter_dropout: residual must have x's shape, dtype and "
                         f"device, got {tuple(residual.shape)} {residual.dtype}")
    return _CounterDropout.apply(x, residual, p, rng, stream)
