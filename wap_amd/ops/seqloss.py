"""The probability of given tokens, and the losses on it that train a decoder
past teacher forcing.

- ``token_logprob`` — log p(y) under rows of logits: what scores hypotheses
  and makes the ``old_logp`` / ``ref_logp`` that the losses take.
- ``policy_loss`` — the clipped policy loss on sampled tokens, with a KL term
  towards a reference.
- ``preference_loss`` — the paired-log-ratio loss on a preferred and a
  rejected sequence.

Conventions are those of ``models.masked_ce``: logits [B,T,K], tokens y [B,T],
weights mask [B,T], loss = sum(mask * l) / max(sum(mask), 1).  A token of
weight 0 is not looked at (its logits may hold anything) and gets a zero
gradient.  A token outside [0, K) that counts makes the result NaN, and its
row's gradient too, unless the upstream gradient of its log-probability is 0
(whoever replaced the NaN depends on nothing there).

The exponentials of a row are f32; their sum and what follows it (logarithm,
ratio, the comparison with the clip's borders, sums over tokens) are f64, since
an error of 1e-7 there can move a token across a border and a gain is a small
difference of long sums.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import op_eager, use_hip
from .functional import _up


def _hip(t: Tensor) -> bool:
    return use_hip(t) and not op_eager("seqloss")


def _live(w: Optional[Tensor], y: Tensor) -> Tensor:
    return torch.ones_like(y, dtype=torch.bool) if w is None else w != 0


def _rows(logits: Tensor, y: Tensor, w: Optional[Tensor]):
    """(logp f64, exponentials, their sum f64, safe token, live, inside) —
    eager."""
    live = _live(w, y)
    k = logits.shape[-1]
    inside = (y >= 0) & (y < k)
    at = torch.where(inside & live, y, 0)
    x = torch.where(live.unsqueeze(-1), _up(logits), 0.0)
    top = x.amax(dim=-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(dim=-1, keepdim=True, dtype=torch.float64)
    logp = (x.gather(-1, at.unsqueeze(-1)).double() - top.double()
            - torch.log(total)).squeeze(-1)
    logp = torch.where(inside, logp, float("nan"))
    return torch.where(live, logp, 0.0), e, total, at, live, inside


def _rows_grad(logits: Tensor, e: Tensor, total: Tensor, at: Tensor,
               live: Tensor, inside: Tensor, coef: Tensor) -> Tensor:
    """coef * (1[k = y] - p), zeros in rows that do not count, NaN for a token
    outside [0, K) that anything depends on — eager."""
    coef = torch.where(inside | (coef == 0), coef, float("nan"))
    d = e * (-coef.unsqueeze(-1) / total).to(e.dtype)
    d.scatter_add_(-1, at.unsqueeze(-1), coef.unsqueeze(-1).to(e.dtype))
    return torch.where(live.unsqueeze(-1), d, 0.0).to(logits.dtype)


class _TokenLogprob(torch.autograd.Function):
    """Eager form, like the two below (the HIP path has its own nodes)."""

    @staticmethod
    def forward(ctx, logits: Tensor, y: Tensor, w: Optional[Tensor]) -> Tensor:
        ctx.save_for_backward(logits, y, w)
        return _rows(logits, y, w)[0].to(_up(logits).dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp: Tensor):
        logits, y, w = ctx.saved_tensors
        _, *rows = _rows(logits, y, w)
        return _rows_grad(logits, *rows, dlogp.double()), None, None


def _policy_terms(logp, old, adv, ref, lo, hi, beta):
    """(loss, d loss / d logp) of every token, f64."""
    adv = adv.double()
    ratio = torch.exp(logp - old.double())
    # an advantage of 0 is worth nothing, however far the ratio is off
    free = torch.where((adv == 0) & ~ratio.isnan(), 0.0, ratio * adv)
    clipped = ratio.clamp(1.0 - lo, 1.0 + hi) * adv
    on = ~(free > clipped)
    loss, slope = -torch.where(on, free, clipped), -torch.where(on, free, 0.0)
    if ref is not None and beta != 0:
        gap = ref.double() - logp
        e = torch.exp(gap)
        # far out the rest is lost beside e, and infinity less itself is none
        loss = loss + beta * torch.where(gap > 64, e, e - gap - 1.0)
        slope = slope + beta * (1.0 - e)
    return loss, slope


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, y, w, old, adv, ref, lo, hi, beta):
        ctx.set_materialize_grads(False)
        logp, _, _, _, live, _ = _rows(logits, y, w)
        l, slope = _policy_terms(logp, old, adv, ref, lo, hi, beta)
        share = w.double() / w.double().sum().clamp_min(1.0)
        loss = torch.where(live, share * l, 0.0).sum().to(_up(logits).dtype)
        coef = torch.where(live, share * slope, 0.0)
        ctx.save_for_backward(logits, y, w, coef)
        logp = logp.to(_up(logits).dtype)
        ctx.mark_non_differentiable(logp)
        return loss, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, up: Optional[Tensor], _):
        none = (None,) * 8
        if up is None:
            return None, *none
        logits, y, w, coef = ctx.saved_tensors
        _, *rows = _rows(logits, y, w)
        return _rows_grad(logits, *rows, coef * up.double()), *none


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, y, w, ref, beta, eps):
        ctx.set_materialize_grads(False)
        logp, _, _, _, live, _ = _rows(logits, y, w)
        gain = torch.where(live, w.double() * (logp - ref.double()), 0.0).sum(1)
        pairs = logits.shape[0] // 2
        m = beta * (gain[:pairs] - gain[pairs:])
        soft = torch.log1p(torch.exp(-m.abs()))
        # a term of coefficient 0 is none, not 0 times an infinite one: the
        # margin is infinite where a token has been ruled out
        each = torch.zeros_like(m)
        if eps < 1:
            each = each + (1 - eps) * (soft + (-m).clamp_min(0))
        if eps > 0:
            each = each + eps * (soft + m.clamp_min(0))
        loss = each.mean()
        slope = beta * (eps * torch.sigmoid(m)
                        - (1 - eps) * torch.sigmoid(-m)) / pairs
        dt = _up(logits).dtype
        margin = m.to(dt)
        ctx.save_for_backward(logits, y, w, torch.cat([slope, -slope]))
        ctx.mark_non_differentiable(margin)
        return loss.to(dt), margin

    @staticmethod
    @once_differentiable
    def backward(ctx, up: Optional[Tensor], _):
        none = (None,) * 5
        if up is None:
            return None, *none
        logits, y, w, seq = ctx.saved_tensors
        _, *rows = _rows(logits, y, w)
        coef = w.double() * seq.unsqueeze(1) * up.double()
        return _rows_grad(logits, *rows, coef), *none


def _check(logits: Tensor, y: Tensor, mask: Optional[Tensor], what: str):
    """Checked and laid out: (logits, y, weights)."""
    if logits.dim() != 3 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must be [B, T, K], got {tuple(logits.shape)}")
    if not logits.is_floating_point():
        raise TypeError(f"{what}: logits must be floating point, got {logits.dtype}")
    if y.is_floating_point() or y.dtype == torch.bool or y.is_complex():
        raise TypeError(f"{what}: y must hold whole numbers, got {y.dtype}")
    if tuple(y.shape) != tuple(logits.shape[:2]) or y.device != logits.device:
        raise ValueError(f"{what}: y must be {tuple(logits.shape[:2])} on "
                         f"{logits.device}, got {tuple(y.shape)} on {y.device}")
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        logits = logits.contiguous()
    return (logits, y.long().contiguous(),
            _per_token(mask, logits, what, "mask"))


def _per_token(t: Optional[Tensor], logits: Tensor, what: str, name: str):
    """A constant [B,T] in f32 (f64 beside f64 logits), contiguous."""
    if t is None:
        return None
    if tuple(t.shape) != tuple(logits.shape[:2]) or t.device != logits.device:
        raise ValueError(f"{what}: {name} must be {tuple(logits.shape[:2])} on "
                         f"{logits.device}, got {tuple(t.shape)} on {t.device}")
    return t.detach().to(_up(logits[:0]).dtype).contiguous()


def token_logprob(logits: Tensor, y: Tensor, mask: Optional[Tensor] = None) -> Tensor:
    """log p(y)[B,T] (f32) of tokens y[B,T] under logits[B,T,K]; 0 where
    mask[B,T] is 0.  Differentiable in logits."""
    if logits.numel() > 0 and _hip(logits):
        from . import ext
        return ext.require().token_logprob(logits, y, mask)
    logits, y, w = _check(logits, y, mask, "token_logprob")
    if logits.numel() == 0:
        return logits.sum(dim=-1).to(_up(logits).dtype)
    return _TokenLogprob.apply(logits, y, w)


def policy_loss(
    logits: Tensor, y: Tensor, mask: Tensor, old_logp: Tensor,
    advantage: Tensor, ref_logp: Optional[Tensor] = None,
    clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
) -> Tuple[Tensor, Tensor]:
    """(loss, logp[B,T]) of the clipped policy loss on sampled tokens y::

        r    = exp(logp - old_logp)
        l    = -min(r * A, clip(r, 1 - clip_low, 1 + clip_high) * A)
             + kl_coef * (exp(ref_logp - logp) - (ref_logp - logp) - 1)
        loss = sum(mask * l) / max(sum(mask), 1)

    ``advantage`` A is [B,T], or [B] for one value a sequence.  ``old_logp``,
    ``ref_logp`` (None, or kl_coef 0: no KL term) and A are constants; logp is returned for
    monitoring, without a gradient.  Differentiable in logits; where a border
    of the clip is met exactly the unclipped side counts.

    Memory: with a gradient wanted, the call keeps a second tensor of the size
    of logits (their gradient for an upstream gradient of one) until the
    backward pass.  Another upstream gradient, a second walk over a kept graph
    and a backward pass captured apart from its forward pass read the logits
    and write the gradient once more."""
    what = "policy_loss"
    if mask is None:
        raise ValueError(f"{what}: mask is required")
    if logits.numel() == 0:
        raise ValueError(f"{what}: no tokens: logits are {tuple(logits.shape)}")
    if not (0.0 <= clip_low and 0.0 <= clip_high):
        raise ValueError(f"{what}: clip borders must be >= 0, got "
                         f"{clip_low}, {clip_high}")
    if _hip(logits):
        from . import ext
        return ext.require().policy_loss(logits, y, mask, old_logp, advantage,
                                         ref_logp, clip_low, clip_high, kl_coef)
    logits, y, w = _check(logits, y, mask, what)
    if advantage.dim() == 1 and advantage.shape[0] == logits.shape[0]:
        advantage = advantage.unsqueeze(1).expand(logits.shape[:2])
    if tuple(advantage.shape) != tuple(y.shape) or advantage.device != logits.device:
        raise ValueError(f"{what}: advantage must be {tuple(y.shape)} or "
                         f"{(y.shape[0],)} on {logits.device}, got "
                         f"{tuple(advantage.shape)} on {advantage.device}")
    old = _per_token(old_logp, logits, what, "old_logp")
    ref = _per_token(ref_logp, logits, what, "ref_logp")
    return _PolicyLoss.apply(logits, y, w, old, advantage.detach().to(w.dtype),
                             ref, float(clip_low), float(clip_high),
                             float(kl_coef))


def preference_loss(
    logits: Tensor, y: Tensor, mask: Tensor, ref_logp: Tensor,
    beta: float = 0.1, label_smoothing: float = 0.0,
) -> Tuple[Tensor, Tensor]:
    """(loss, margin[P]) of P pairs of sequences: rows 0..P-1 of logits
    [2P,T,K] are the preferred ones, rows P..2P-1 the rejected::

        gain_b   = sum_t mask * (logp - ref_logp)
        margin_i = beta * (gain_i - gain_{P+i})
        loss     = mean_i( -(1 - s) log sigmoid(margin_i)
                           - s log sigmoid(-margin_i) ),  s = label_smoothing

    ``ref_logp`` [2P,T] is the reference's ``token_logprob``, a constant; the
    margin is returned without a gradient.  Differentiable in logits.  A token
    of probability 0 makes its pair's margin infinite and the loss what the
    formula tends to: nothing of that pair where the token is rejected and s
    is 0."""
    what = "preference_loss"
    if mask is None:
        raise ValueError(f"{what}: mask is required")
    if ref_logp is None:
        raise ValueError(f"{what}: ref_logp is required")
    if logits.numel() == 0 or logits.shape[0] % 2:
        raise ValueError(f"{what}: sequences come in pairs: logits are "
                         f"{tuple(logits.shape)}")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"{what}: label_smoothing must be in [0, 1], got "
                         f"{label_smoothing}")
    if _hip(logits):
        from . import ext
        return ext.require().preference_loss(logits, y, mask, ref_logp, beta,
                                             label_smoothing)
    logits, y, w = _check(logits, y, mask, what)
    ref = _per_token(ref_logp, logits, what, "ref_logp")
    return _PreferenceLoss.apply(logits, y, w, ref, float(beta),
                                 float(label_smoothing))
