"""64-bit values of the sequence operators and elementwise error bounds.

Plain formulas in float64, apart from wap_amd.ops.  Each ``*_bound`` follows
the operator's roundings in f32 (unit U = 2^-24) through the same formula, so
that a tolerance is a sum of errors that can happen, plus half a step of the
type that the result is stored in."""

import math

import torch

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(v, dtype):
    """Half a step of ``dtype`` at v, and of its smallest numbers."""
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38,
            torch.float32: 1e-38}[dtype]
    return v.abs() * (torch.finfo(dtype).eps / 2) + tiny


def assert_within(got, want, bound, what=""):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    bound = bound.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, torch.zeros_like(got), (got - want).abs())
    bad = ~(off <= bound)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
        f"{float((off / bound.clamp_min(1e-300)).nan_to_num(math.inf).max()):.2f} "
        f"of the bound")


# ------------------------------------------------------ gated recurrence

# Roundings of one step, in units of U: two exponential-type functions of at
# most 2 ulp (4 U) whose argument may carry |x| U (|x| < 12 in these tests),
# a reciprocal, three products and sums.
STEP = 32 * U


def scan(g, h0, mask, dh=None, dlast=None):
    """f64 results and their bounds: dict of name -> (value, bound)."""
    g = g.detach().double().cpu()
    b, t, d = g.shape[0], g.shape[1], g.shape[2] // 2
    z, n = torch.sigmoid(g[..., :d]), torch.tanh(g[..., d:])
    zc = torch.sigmoid(-g[..., :d])
    on = (torch.ones(b, t, 1, dtype=torch.bool) if mask is None
          else mask.detach().cpu()[..., None] > 0)
    h = torch.zeros(b, d, dtype=torch.float64) if h0 is None else h0.detach().double().cpu()
    e = torch.zeros_like(h)
    past, past_e, hs, es = [], [], [], []
    for i in range(t):
        past.append(h)
        past_e.append(e)
        new_e = z[:, i] * e + STEP * (z[:, i] * h.abs() + zc[:, i] * n[:, i].abs())
        h = torch.where(on[:, i], zc[:, i] * n[:, i] + z[:, i] * h, h)
        e = torch.where(on[:, i], new_e, e)
        hs.append(h)
        es.append(e)
    out = {"h": (torch.stack(hs, 1), torch.stack(es, 1)), "last": (h, e)}
    if dh is None and dlast is None:
        return out
    up = torch.zeros(b, t, d, dtype=torch.float64) if dh is None else dh.detach().double().cpu()
    c = torch.zeros_like(h) if dlast is None else dlast.detach().double().cpu()
    ec = torch.zeros_like(h)
    dg, eg = torch.zeros_like(g), torch.zeros_like(g)
    for i in reversed(range(t)):
        c = c + up[:, i]
        ec = ec + 2 * U * (c.abs() + up[:, i].abs())
        zi, qi, ni, hi, ei = z[:, i], zc[:, i], n[:, i], past[i], past_e[i]
        slope, nn = zi * qi, 1 - ni * ni
        gz, gn = c * (hi - ni) * slope, c * qi * nn
        egz = (ec * (hi - ni).abs() * slope + c.abs() * slope * (ei + STEP * (hi.abs() + ni.abs()))
               + STEP * gz.abs())
        egn = ec * qi * nn + c.abs() * qi * STEP * (nn + 2 * ni * ni) + STEP * gn.abs()
        dg[:, i] = torch.where(on[:, i], torch.cat([gz, gn], -1), 0.0)
        eg[:, i] = torch.where(on[:, i], torch.cat([egz, egn], -1), 0.0)
        ec = torch.where(on[:, i], zi * ec + STEP * (zi * c).abs(), ec)
        c = torch.where(on[:, i], zi * c, c)
    out["dg"], out["dh0"] = (dg, eg), (c, ec)
    return out


# ------------------------------------------------------ token probabilities

def rows(logits, y, w=None):
    """(logp, bound of its error before rounding, p, relative bound of p)."""
    x = logits.detach().double().cpu()
    y = y.cpu()
    k = x.shape[-1]
    live = torch.ones(y.shape, dtype=torch.bool) if w is None else w.cpu() != 0
    x = torch.where(live[..., None], x, 0.0)
    inside = (y >= 0) & (y < k)
    at = torch.where(inside, y, 0)
    logp_all = torch.log_softmax(x, -1)
    p = logp_all.exp()
    logp = logp_all.gather(-1, at[..., None])[..., 0]
    logp = torch.where(inside, logp, math.nan)
    logp = torch.where(live, logp, 0.0)
    d = (x.amax(-1, keepdim=True) - x).clamp(max=200.0)
    # an exponential of d: its argument's rounding d U, 4 U of its own;
    # a chain of at most K / 64 additions (64 lanes share a row) and a tree
    each = (d + 6) * U
    total = (p * each).sum(-1, keepdim=True) + (min(k / 64, 600) + 16) * U
    return logp, total[..., 0], p, each + total + 4 * U, at, live


def rows_grad(coef, ecoef, p, ep, at, live):
    one = torch.zeros_like(p).scatter_(-1, at[..., None], 1.0)
    c = coef[..., None]
    d = torch.where(live[..., None], c * (one - p), 0.0)
    bound = (c.abs() * p * ep + ecoef[..., None] * (one + p)
             + 4 * U * c.abs() * (one + p))
    return d, torch.where(live[..., None], bound, 0.0)


def policy(logits, y, w, old, adv, ref, lo, hi, beta, up=1.0):
    logp, elog, p, ep, at, live = rows(logits, y, w)
    w, old, adv = (v.detach().double().cpu() for v in (w, old, adv))
    adv = adv[:, None].expand(w.shape) if adv.dim() == 1 else adv
    ratio = torch.exp(logp - old)
    kept = ratio.clamp(1 - lo, 1 + hi)
    free, clipped = ratio * adv, kept * adv
    on = ~(free > clipped)
    loss, slope = -torch.where(on, free, clipped), -torch.where(on, free, 0.0)
    err = free.abs()
    if ref is not None:
        gap = ref.detach().double().cpu() - logp
        loss = loss + beta * (gap.exp() - gap - 1)
        slope = slope + beta * (1 - gap.exp())
        err = err + beta * (gap.exp() + 1)
    share = w / w.sum().clamp_min(1.0)
    loss = torch.where(live, share * loss, 0.0)
    coef = torch.where(live, up * share * slope, 0.0)
    ecoef = abs(up) * share * err * 2 * elog + 2 * U * coef.abs()
    eloss = (share * err * 2 * elog).sum()
    near = torch.minimum((ratio - (1 - lo)).abs(), (ratio - (1 + hi)).abs())
    clear = bool((near[live] > 4 * (ratio * elog)[live]).all())
    d, ed = rows_grad(coef, ecoef, p, ep, at, live)
    return loss.sum(), eloss, logp, elog, d, ed, clear


def preference(logits, y, w, ref, beta, eps, up=1.0):
    logp, elog, p, ep, at, live = rows(logits, y, w)
    w, ref = w.detach().double().cpu(), ref.detach().double().cpu()
    gain = torch.where(live, w * (logp - ref), 0.0).sum(1)
    egain = torch.where(live, w * elog, 0.0).sum(1)
    half = gain.shape[0] // 2
    m = beta * (gain[:half] - gain[half:])
    em = beta * (egain[:half] + egain[half:])
    ls = torch.nn.functional.logsigmoid
    loss = -((1 - eps) * ls(m) + eps * ls(-m)).mean()
    slope = beta * (eps * torch.sigmoid(m) - (1 - eps) * torch.sigmoid(-m)) / half
    # both sigmoids' slope is at most 1/4, and at most themselves
    eslope = beta / half * em * torch.minimum(
        torch.full_like(m, 0.25), (1 - eps) * torch.sigmoid(-m) + eps * torch.sigmoid(m)) * 2
    seq, eseq = torch.cat([slope, -slope])[:, None], torch.cat([eslope, eslope])[:, None]
    coef = torch.where(live, up * w * seq, 0.0)
    ecoef = torch.where(live, abs(up) * w * eseq, 0.0) + 4 * U * coef.abs()
    d, ed = rows_grad(coef, ecoef, p, ep, at, live)
    return loss, em.mean(), m, em, d, ed


# ------------------------------------------------------ dropout

def draws(n, seed, step, stream):
    """16-bit draws by Python's whole numbers."""
    out = []
    low = 0xFFFFFFFF
    for group in range((n + 7) // 8):
        c = [group & low, (stream << 8) | (group >> 32), step & low, (step >> 32) & low]
        k = [seed & low, (seed >> 32) & low]
        for _ in range(7):
            p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(q >> 32) ^ c[1] ^ k[0], q & low, (p >> 32) ^ c[3] ^ k[1], p & low]
            k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
        for v in c:
            out += [v & 0xFFFF, v >> 16]
    return torch.tensor(out[:n])


def dropout(x, p, seed, step, stream, residual=None):
    """x, residual contiguous -> (value, bound, kept)."""
    limit = math.floor(p * 65536 + 0.5)
    keep = (draws(x.numel(), seed, step, stream) >= limit).view(x.shape)
    scale = 65536 / (65536 - limit) if limit < 65536 else 0.0
    v = torch.where(keep, x.detach().double().cpu() * scale, 0.0)
    bound = 3 * U * v.abs()
    if residual is not None:
        r = residual.detach().double().cpu()
        v = v + r
        bound = bound + U * (v.abs() + r.abs())
    return v, bound + half_step(v, x.dtype), keep
