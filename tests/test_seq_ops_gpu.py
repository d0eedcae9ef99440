"""Sequence operators' HIP kernels against the 64-bit formulas, with the
bounds of tests/seq_oracle.py (sums of roundings, half a step of the type)."""

import math

import pytest
import torch

import seq_oracle as oracle
from seq_oracle import DTYPES, U, assert_within, half_step

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _hip_backend():
    from wap_amd import ops
    from wap_amd.ops import ext
    assert ext.available(), "HIP extension must be loadable on the GPU box"
    ops.set_backend("hip")
    yield
    ops.set_backend("auto")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def drain():
    """Waits for the stream by a copy to the host."""
    torch.zeros(1, device=DEV).item()


# ------------------------------------------------------ gated recurrence

def _scan_inputs(b, t, d, dtype, seed, mask=False, start=True):
    r = gen(seed)
    g = torch.randn(b, t, 2 * d, generator=r) * 1.5
    g[..., :d] += 2.0
    m = None
    if mask:
        m = (torch.rand(b, t, generator=r) < 0.7).float()
        m[-1] = 0
    h0 = torch.randn(b, d, generator=r) if start else None
    dh = torch.randn(b, t, d, generator=r)
    dl = torch.randn(b, d, generator=r)
    to = lambda v, dt=torch.float32: None if v is None else v.to(dt).to(DEV)  # noqa: E731
    return to(g, dtype), to(h0), to(m), to(dh, dtype), to(dl)


def _check_scan(g, h0, m, dh, dl, dtype):
    from wap_amd import ops
    g = g.requires_grad_()
    leaves = (g,)
    if h0 is not None:
        h0 = h0.requires_grad_()
        leaves += (h0,)
    h, last = ops.gated_scan(g, h0, m)
    assert h.dtype == dtype and last.dtype == torch.float32
    outs, ups = [], []
    for o, u in ((h, dh), (last, dl)):
        if u is not None:
            outs.append(o)
            ups.append(u)
    grads = torch.autograd.grad(outs, leaves, ups)
    want = oracle.scan(g, h0, m, dh, dl)
    for name, got in [("h", h), ("last", last), ("dg", grads[0])] + (
            [("dh0", grads[1])] if h0 is not None else []):
        v, e = want[name]
        assert_within(got, v, e + half_step(v, got.dtype), name)
    return h, last, grads


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,d", [
    (1, 1, 1), (3, 1, 64), (2, 2, 7), (5, 17, 33), (2, 63, 64), (2, 64, 65),
    (1, 65, 128), (3, 129, 130), (2, 256, 256), (1, 257, 66), (2, 300, 10),
    (1, 1025, 129), (1, 2500, 34), (70, 3, 3), (1, 5, 2051), (16, 200, 256),
])
def test_scan(b, t, d, dtype):
    _check_scan(*_scan_inputs(b, t, d, dtype, b + t + d), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,d", [(2, 1, 5), (3, 130, 64), (2, 700, 129), (4, 33, 256)])
@pytest.mark.parametrize("start", [False, True])
def test_scan_masked(b, t, d, dtype, start):
    _check_scan(*_scan_inputs(b, t, d, dtype, t, mask=True, start=start), dtype)


@pytest.mark.parametrize("which", ["dh", "dlast"])
def test_scan_one_upstream(which):
    g, h0, m, dh, dl = _scan_inputs(2, 150, 40, torch.float32, 1, mask=True)
    dh, dl = (dh, None) if which == "dh" else (None, dl)
    _check_scan(g, h0, m, dh, dl, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_long_memory(dtype):
    """Gates close to one: the state holds thousands of steps."""
    g, h0, m, dh, dl = _scan_inputs(1, 3000, 16, dtype, 2)
    g[..., :16] += 6
    _check_scan(g, h0, m, dh, dl, dtype)


def test_scan_gates_at_their_ends():
    """z exactly 0 or 1 in f32, infinite gates: no NaN, state kept or replaced."""
    d = 8
    g = torch.zeros(1, 6, 2 * d, device=DEV)
    g[0, :, :d] = torch.tensor([200., -200., 60., -60., math.inf, -math.inf], device=DEV)[:, None]
    g[0, :, d:] = torch.tensor([1., 50., -50., math.inf, -math.inf, 0.5], device=DEV)[:, None]
    h0 = torch.full((1, d), 0.25, device=DEV)
    h, last, _ = _check_scan(g, h0, None, torch.ones(1, 6, d, device=DEV), None, torch.float32)
    assert (h[0, 0] == 0.25).all() and (h[0, 1] == 1).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [5, 400])
def test_scan_strides(t, dtype):
    """Gates and upstream gradients inside wider tensors, at odd places."""
    b, d = 3, 66
    g, h0, m, dh, dl = _scan_inputs(b, t, d, dtype, 3)
    for off in (0, 1, 3):
        wide = torch.zeros(t + 2, b, 2 * d + 5, device=DEV, dtype=dtype)
        wide[1:-1, :, off:off + 2 * d] = g.detach().transpose(0, 1)
        view = wide[1:-1, :, off:off + 2 * d].transpose(0, 1)
        up = torch.zeros(b, t, d + 3, device=DEV, dtype=dtype)
        up[..., off:off + d] = dh
        _check_scan(view.detach(), h0.detach(), None, up[..., off:off + d], dl, dtype)
    last_first = g.detach().permute(2, 0, 1).contiguous().permute(1, 2, 0)
    _check_scan(last_first, h0.detach(), None, dh[:, :1].expand(b, t, d), dl, dtype)


@pytest.mark.parametrize("t", [40, 700])
def test_scan_masked_gates_are_not_looked_at(t):
    from wap_amd import ops
    g, h0, m, dh, dl = _scan_inputs(3, t, 70, torch.bfloat16, 4, mask=True)
    dirty = g.clone()
    dirty[m == 0] = math.nan
    outs = []
    for x in (g, dirty):
        x.requires_grad_()
        h, last = ops.gated_scan(x, h0, m)
        outs.append((h, last, torch.autograd.grad((h, last), x, (dh, dl))[0]))
    for a, c in zip(*outs):
        assert torch.equal(a, c)
    assert (outs[0][2][m == 0] == 0).all()
    assert torch.equal(outs[0][1][-1], h0[-1])


@pytest.mark.parametrize("mask_type", [torch.bool, torch.int64, torch.bfloat16])
def test_scan_mask_types(mask_type):
    from wap_amd import ops
    g, h0, m, *_ = _scan_inputs(2, 30, 8, torch.float32, 5, mask=True)
    want = ops.gated_scan(g, h0, m)
    got = ops.gated_scan(g, h0, m.to(mask_type))
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.parametrize("b,t,d", [(2, 100, 64), (1, 5000, 256), (4, 1500, 130)])
def test_scan_repeats_bit_for_bit(b, t, d):
    from wap_amd import ops
    g, h0, m, dh, dl = _scan_inputs(b, t, d, torch.bfloat16, 6, mask=True)
    g.requires_grad_()
    h0.requires_grad_()
    first = None
    for _ in range(4):
        h, last = ops.gated_scan(g, h0, m)
        now = (h, last, *torch.autograd.grad((h, last), (g, h0), (dh, dl)))
        if first is not None:
            assert all(torch.equal(a, c) for a, c in zip(first, now))
        first = now


def test_scan_is_the_same_cut_anywhere():
    """A sequence walked in two calls, the state carried between them."""
    from wap_amd import ops
    g, h0, *_ = _scan_inputs(2, 900, 64, torch.float32, 7)
    h, last = ops.gated_scan(g, h0)
    for cut in (1, 64, 500, 899):
        a, mid = ops.gated_scan(g[:, :cut], h0)
        c, end = ops.gated_scan(g[:, cut:], mid)
        # f32 in another order: the bound of the recurrence itself
        want = oracle.scan(g, h0, None)
        assert_within(torch.cat([a, c], 1), want["h"][0], want["h"][1] + half_step(want["h"][0], torch.float32))
        assert_within(end, want["last"][0], want["last"][1])


def test_scan_offsets_past_32_bits():
    from wap_amd import ops
    b, t, d = 12000, 3, 32768
    g = torch.empty(b, t, 2 * d, device=DEV, dtype=torch.bfloat16)
    part = [_scan_inputs(2, t, d, torch.bfloat16, s) for s in (8, 9)]
    g[:2], g[-2:] = part[0][0], part[1][0]
    g[2:-2] = 0
    g.requires_grad_()
    h, last = ops.gated_scan(g)
    dh = torch.zeros_like(h)
    dh[:2], dh[-2:] = part[0][3], part[1][3]
    dg, = torch.autograd.grad(h, g, dh)
    for at, p in ((slice(0, 2), part[0]), (slice(b - 2, b), part[1])):
        want = oracle.scan(p[0], None, None, p[3], None)
        for name, got in (("h", h[at]), ("last", last[at]), ("dg", dg[at])):
            v, e = want[name]
            assert_within(got, v, e + half_step(v, got.dtype), name)
    assert not dg[2:100].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,d", [(1, 1), (80, 256), (7, 33), (1, 4096), (513, 130)])
def test_step(b, d, dtype):
    from wap_amd import ops
    g, h0, *_ = _scan_inputs(b, 1, d, dtype, b + d)
    keep = h0.clone()
    out, new = ops.gated_step(g[:, 0], h0)
    want = oracle.scan(g, h0, None)["last"]
    assert out.dtype == dtype and new.dtype == torch.float32
    assert_within(new, want[0], want[1])
    assert_within(out, want[0], want[1] + half_step(want[0], dtype))
    assert torch.equal(h0, keep)
    wide = torch.zeros(b, 2 * d + 3, device=DEV, dtype=dtype)
    wide[:, 1:-2] = g[:, 0]
    again = ops.gated_step(wide[:, 1:-2], h0)
    assert torch.equal(again[0], out) and torch.equal(again[1], new)


# ------------------------------------------------------ token probabilities

def _loss_inputs(b, t, k, dtype, seed, spread=2.0):
    r = gen(seed)
    logits = (torch.randn(b, t, k, generator=r) * spread).to(dtype)
    y = torch.randint(k, (b, t), generator=r)
    w = (torch.rand(b, t, generator=r) < 0.8).float()
    w[0, 0] = 1
    if b > 1:
        w[-1] = 0
    near = torch.log_softmax(logits.double(), -1).gather(-1, y[..., None])[..., 0]
    old = (near + 0.2 * torch.randn(b, t, generator=r)).float()
    ref = (near + 0.2 * torch.randn(b, t, generator=r)).float()
    adv = torch.randn(b, t, generator=r)
    return tuple(v.to(DEV) for v in (logits, y, w, old, ref, adv))


SIZES = [
    (1, 1, 1), (2, 3, 2), (1, 2, 63), (3, 5, 64), (2, 7, 112), (2, 2, 255),
    (2, 3, 1000), (1, 3, 2048), (2, 2, 2049), (1, 2, 4097), (2, 2, 8192),
    (1, 2, 10007), (1, 2, 16384), (1, 1, 16385), (1, 2, 32768), (1, 2, 50001),
    (1, 1, 65537), (1, 1, 131072), (1, 2, 140001),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,k", SIZES)
def test_token_logprob(b, t, k, dtype):
    from wap_amd import ops
    logits, y, w, *_ = _loss_inputs(b, t, k, dtype, b + t + k)
    logits.requires_grad_()
    up = torch.randn(b, t, generator=gen(1)).to(DEV)
    for mask in (None, w):
        got = ops.token_logprob(logits, y, mask)
        logp, elog, p, ep, at, live = oracle.rows(logits, y, mask)
        assert_within(got, logp, elog + half_step(logp, torch.float32), "logp")
        d, = torch.autograd.grad(got, logits, up)
        c = torch.where(live, up.double().cpu(), 0.0)
        want, bound = oracle.rows_grad(c, torch.zeros_like(c), p, ep, at, live)
        assert_within(d, want, bound + half_step(want, dtype), "dlogits")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,k", SIZES)
def test_policy_loss(b, t, k, dtype):
    from wap_amd import ops
    logits, y, w, old, ref, adv = _loss_inputs(b, t, k, dtype, 7 * b + t + k)
    logits.requires_grad_()
    for use_ref, up in ((True, 1.0), (False, 1.0), (True, 0.25)):
        r = ref if use_ref else None
        want, eloss, logp, elog, d, ed, clear = oracle.policy(
            logits, y, w, old, adv, r, 0.2, 0.3, 0.1, up)
        assert clear, "a token of this test lies at a border of the clip"
        loss, lp = ops.policy_loss(logits, y, w, old, adv, r, clip_low=0.2,
                                   clip_high=0.3, kl_coef=0.1)
        assert_within(loss, want, eloss + U * want.abs() * 2, "loss")
        assert_within(lp, logp, elog + half_step(logp, torch.float32), "logp")
        got, = torch.autograd.grad(loss, logits, torch.tensor(up, device=DEV))
        assert got.dtype == dtype
        assert_within(got, d, ed + half_step(d, dtype), "dlogits")
        with torch.no_grad():
            assert torch.equal(ops.policy_loss(
                logits, y, w, old, adv, r, clip_low=0.2, clip_high=0.3,
                kl_coef=0.1)[0], loss)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,k", [(2 * b, t, k) for b, t, k in SIZES])
def test_preference_loss(b, t, k, dtype):
    from wap_amd import ops
    logits, y, w, _, ref, _ = _loss_inputs(b, t, k, dtype, 5 * b + t + k)
    logits.requires_grad_()
    for eps, up in ((0.0, 1.0), (0.2, 0.5)):
        want, el, m, em, d, ed = oracle.preference(logits, y, w, ref, 0.5, eps, up)
        loss, margin = ops.preference_loss(logits, y, w, ref, beta=0.5, label_smoothing=eps)
        assert_within(loss, want, el + 2 * U * want.abs(), "loss")
        assert_within(margin, m, em + 2 * U * m.abs(), "margin")
        got, = torch.autograd.grad(loss, logits, torch.tensor(up, device=DEV))
        assert got.dtype == dtype
        assert_within(got, d, ed + half_step(d, dtype), "dlogits")


def test_many_rows():
    """More rows than one workgroup's walk over the weights, fractions among them."""
    from wap_amd import ops
    b, t, k = 37, 301, 20
    logits, y, w, old, ref, adv = _loss_inputs(b, t, k, torch.float32, 3)
    w = w * torch.rand(b, t, generator=gen(4)).to(DEV)
    logits.requires_grad_()
    want, el, _, _, d, ed, clear = oracle.policy(logits, y, w, old, adv, ref, 0.2, 0.2, 0.1)
    assert clear
    loss, _ = ops.policy_loss(logits, y, w, old, adv, ref, kl_coef=0.1)
    assert_within(loss, want, el + 2 * U * want.abs())
    got, = torch.autograd.grad(loss, logits)
    assert_within(got, d, ed + half_step(d, torch.float32))
    b = 36
    args = [v[:b].detach() for v in (logits, y, w, ref)]
    args[0].requires_grad_()
    want, el, m, em, d, ed = oracle.preference(*args, 0.1, 0.0)
    loss, margin = ops.preference_loss(*args, beta=0.1)
    assert_within(loss, want, el + 2 * U * want.abs())
    assert_within(margin, m, em + 2 * U * m.abs())
    got, = torch.autograd.grad(loss, args[0])
    assert_within(got, d, ed + half_step(d, torch.float32))


@pytest.mark.parametrize("k", [50, 3000, 70001])
def test_advantage_of_a_sequence(k):
    from wap_amd import ops
    logits, y, w, old, ref, adv = _loss_inputs(3, 4, k, torch.bfloat16, k)
    a = ops.policy_loss(logits, y, w, old, adv[:, 0], ref, kl_coef=0.1)
    c = ops.policy_loss(logits, y, w, old, adv[:, :1].expand(3, 4), ref, kl_coef=0.1)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [112, 2500, 20001, 140001])
def test_loss_strides(k, dtype):
    """Logits as a slice in time, and inside wider rows at an odd place."""
    from wap_amd import ops
    b, t = 2, 3
    logits, y, w, old, ref, adv = _loss_inputs(b, t, k, dtype, k + 1)

    def all_of(x):
        x = x.detach().requires_grad_()
        l1, lp = ops.policy_loss(x, y, w, old, adv, ref, kl_coef=0.1)
        l2, m = ops.preference_loss(x, y, w, ref)
        s = ops.token_logprob(x, y, w)
        return (l1, lp, l2, m, s, torch.autograd.grad(l1, x)[0],
                torch.autograd.grad(l2, x)[0], torch.autograd.grad(s.sum(), x)[0])

    want = all_of(logits)
    longer = torch.full((b, t + 1, k), math.nan, device=DEV, dtype=dtype)
    longer[:, :-1] = logits
    wide = torch.full((b, t, k + 3), math.nan, device=DEV, dtype=dtype)
    wide[..., 1:-2] = logits
    turned = logits.transpose(0, 1).contiguous().transpose(0, 1)
    spread = logits.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    for name, x in (("time", longer[:, :-1]), ("row", wide[..., 1:-2]),
                    ("turned", turned), ("spread", spread)):
        for u, v in zip(want, all_of(x)):
            assert torch.equal(u, v), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [100, 5000, 140001])
def test_masked_rows_may_hold_anything(k, dtype):
    from wap_amd import ops
    logits, y, w, old, ref, adv = _loss_inputs(4, 3, k, dtype, k)
    off = w == 0
    bad = [v.clone() for v in (logits, old, ref, adv)]
    for v in bad:
        v[off] = math.nan
    y2 = torch.where(off, -100, y)
    res = []
    for (x, o, r, a), yy in (((logits, old, ref, adv), y), (bad, y2)):
        x.requires_grad_()
        l1, lp = ops.policy_loss(x, yy, w, o, a, r, kl_coef=0.1)
        l2, m = ops.preference_loss(x, yy, w, r)
        s = ops.token_logprob(x, yy, w)
        res.append((l1, lp, l2, m, s, torch.autograd.grad(l1, x)[0],
                    torch.autograd.grad(l2, x)[0], torch.autograd.grad(s.sum(), x)[0]))
    for u, v in zip(*res):
        assert torch.equal(u, v)
    for d in res[1][-3:]:
        assert (d[off] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [100, 5000, 140001])
def test_forbidden_tokens(k, dtype):
    """Logits of minus infinity and of the type's lowest value: probability
    and gradient zero, the others as if those were not there."""
    from wap_amd import ops
    logits, y, w, old, ref, adv = _loss_inputs(2, 3, k, dtype, k)
    w = torch.ones_like(w)
    y = torch.zeros_like(y)
    for low in (-math.inf, torch.finfo(dtype).min):
        x = logits.clone()
        x[..., 1::2] = low
        x.requires_grad_()
        s = ops.token_logprob(x, y)
        d, = torch.autograd.grad(s.sum(), x)
        assert (d[..., 1::2] == 0).all()
        logp, elog, p, ep, at, live = oracle.rows(x[..., ::2], y)
        assert_within(s, logp, elog + half_step(logp, torch.float32))
        one = torch.ones_like(logp)
        want, bound = oracle.rows_grad(one, 0 * one, p, ep, at, live)
        assert_within(d[..., ::2], want, bound + half_step(want, dtype))


@pytest.mark.parametrize("k", [100, 5000, 140001])
def test_nan_and_infinities_are_loud(k):
    from wap_amd import ops
    logits, y, w, old, ref, adv = _loss_inputs(2, 3, k, torch.float32, k)
    w = torch.ones_like(w)
    for value in (math.nan, math.inf):
        for at in (0, k // 2, k - 1):
            x = logits.clone()
            x[1, 1, at] = value
            s = ops.token_logprob(x, y)
            assert torch.isnan(s[1, 1]) and torch.isfinite(s[0]).all()
            assert torch.isnan(ops.policy_loss(x, y, w, old, adv)[0])
            assert torch.isnan(ops.preference_loss(x, y, w, ref)[0])
    x = logits.clone()
    x[0, 0] = -math.inf
    assert torch.isnan(ops.token_logprob(x, y)[0, 0])
    for bad in (-1, k, 1 << 40):
        y2 = y.clone()
        y2[1, 2] = bad
        s = ops.token_logprob(logits, y2)
        assert torch.isnan(s[1, 2]) and torch.isfinite(s[0]).all()
        assert torch.isnan(ops.policy_loss(logits, y2, w, old, adv)[0])


def test_large_logits():
    """Far from zero and far from each other: the maximum is taken off first."""
    from wap_amd import ops
    for k in (120, 40000):
        logits, y, w, *_ = _loss_inputs(2, 3, k, torch.float32, k)
        x = logits * 3000 + 1e6
        s = ops.token_logprob(x, y)
        logp, elog, *_ = oracle.rows(x, y)
        assert_within(s, logp, elog + half_step(logp, torch.float32))


@pytest.mark.parametrize("k", [112, 5000, 140001])
def test_policy_backward_twice(k):
    """A kept graph, other upstream gradients: results stay the caller's."""
    from wap_amd import ops
    logits, y, w, old, ref, adv = _loss_inputs(3, 4, k, torch.float32, 2)
    x = logits.requires_grad_()
    loss, _ = ops.policy_loss(x, y, w, old, adv, ref, kl_coef=0.1)
    first, = torch.autograd.grad(loss, x, torch.tensor(2.0, device=DEV), retain_graph=True)
    kept = first.clone()
    second, = torch.autograd.grad(loss, x, retain_graph=True)
    third, = torch.autograd.grad(loss, x, torch.tensor(0.0, device=DEV), retain_graph=True)
    assert torch.equal(first, kept)
    # scaling by two is exact
    assert torch.equal(first, 2 * second)
    assert (third == 0).all()
    nan, = torch.autograd.grad(loss, x, torch.tensor(math.nan, device=DEV))
    assert torch.isnan(nan[w > 0]).all() and (nan[w == 0] == 0).all()


def test_policy_loss_in_a_sum_of_losses():
    from wap_amd import ops
    logits, y, w, old, ref, adv = _loss_inputs(2, 3, 60, torch.float32, 2)
    x = logits.requires_grad_()
    parts = []
    for f in (lambda: ops.policy_loss(x, y, w, old, adv, ref, kl_coef=0.1)[0],
              lambda: ops.preference_loss(x, y, w, ref)[0],
              lambda: ops.token_logprob(x, y, w).sum()):
        parts.append(torch.autograd.grad(f(), x)[0])
    total = (ops.policy_loss(x, y, w, old, adv, ref, kl_coef=0.1)[0]
             + ops.preference_loss(x, y, w, ref)[0] + ops.token_logprob(x, y, w).sum())
    total.backward()
    # two f32 sums of three parts, in whichever order
    size = sum(p.abs() for p in parts)
    assert_within(x.grad, sum(p.double() for p in parts), 4 * U * size)


def test_loss_offsets_past_32_bits():
    from wap_amd import ops
    b, t, k = 2, 17000, 70000
    logits = torch.zeros(b, t, k, device=DEV, dtype=torch.bfloat16)
    y = torch.zeros(b, t, dtype=torch.long, device=DEV)
    w = torch.zeros(b, t, device=DEV)
    old = torch.zeros(b, t, device=DEV)
    some = _loss_inputs(2, 3, k, torch.bfloat16, 1)
    for i in range(2):
        logits[i, -3:], y[i, -3:], w[i, -3:], old[i, -3:] = (
            some[0][i], some[1][i], 1.0, some[3][i])
    logits.requires_grad_()
    adv = torch.ones(b, device=DEV)
    one = torch.ones(2, 3, device=DEV)
    args = (some[0], some[1], one, some[3], one, None, 0.2, 0.2, 0.0)
    want, el, logp, elog, d, ed, clear = oracle.policy(*args)
    assert clear
    loss, lp = ops.policy_loss(logits, y, w, old, adv)
    assert_within(loss, want, el + 2 * U * want.abs())
    assert_within(lp[:, -3:], logp, elog + half_step(logp, torch.float32))
    got, = torch.autograd.grad(loss, logits)
    assert_within(got[:, -3:], d, ed + half_step(d, torch.bfloat16))
    assert not got[:, :-3].any()
    del got
    got, = torch.autograd.grad(ops.token_logprob(logits, y, w).sum(), logits)
    logp, elog, p, ep, at, live = oracle.rows(some[0], some[1])
    c = torch.ones_like(logp)
    v, bound = oracle.rows_grad(c, 0 * c, p, ep, at, live)
    assert_within(got[:, -3:], v, bound + half_step(v, torch.bfloat16))


# ------------------------------------------------------ dropout

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 255, 2048, 5001])
@pytest.mark.parametrize("seed,step,stream", [(0, 0, 0), (-9, 2 ** 40 + 3, 2 ** 24 - 1)])
def test_dropout(n, dtype, seed, step, stream):
    from wap_amd import ops
    x = (torch.randn(n, generator=gen(n)) + 4).to(dtype).to(DEV).requires_grad_()
    res = torch.randn(n, generator=gen(n + 1)).to(dtype).to(DEV).requires_grad_()
    dy = (torch.randn(n, generator=gen(n + 2)) + 4).to(dtype).to(DEV)
    for rng in ((seed, step), torch.tensor([seed, step], device=DEV)):
        for p in (0.25, 0.9):
            y = ops.counter_dropout(x, p, rng, stream)
            want, bound, keep = oracle.dropout(x, p, seed, step, stream)
            assert torch.equal((y != 0).cpu(), keep)
            assert_within(y, want, bound)
            y = ops.counter_dropout(x, p, rng, stream, res)
            want, bound, _ = oracle.dropout(x, p, seed, step, stream, res)
            assert_within(y, want, bound)
            dx, dr = torch.autograd.grad(y, (x, res), dy)
            want, bound, _ = oracle.dropout(dy, p, seed, step, stream)
            assert_within(dx, want, bound)
            assert torch.equal(dr, dy)
    assert torch.equal(ops.counter_dropout(x, 0.0, (1, 1)), x)
    assert (ops.counter_dropout(x, 1.0, (1, 1)) == 0).all()


def test_dropout_nan_dropped_and_layouts():
    from wap_amd import ops
    x = torch.full((2, 24, 5, 7), math.nan, device=DEV, dtype=torch.bfloat16)
    x = x.to(memory_format=torch.channels_last)
    y = ops.counter_dropout(x, 0.5, (0, 0))
    assert y.is_contiguous(memory_format=torch.channels_last)
    keep = oracle.dropout(torch.ones(x.numel()), 0.5, 0, 0, 0)[2]
    flat = y.permute(0, 2, 3, 1).reshape(-1).cpu()
    assert torch.equal(torch.isnan(flat), keep) and (flat[~keep] == 0).all()
    # at an odd place of a larger buffer, and not dense
    buf = torch.randn(1000, device=DEV).bfloat16()
    for off in (1, 2, 3, 5):
        got = ops.counter_dropout(buf[off:off + 801], 0.5, (3, 3))
        assert torch.equal(got, ops.counter_dropout(buf[off:off + 801].clone(), 0.5, (3, 3)))
    sq = torch.randn(40, 50, device=DEV)
    assert torch.equal(ops.counter_dropout(sq.t(), 0.5, (3, 3)),
                       ops.counter_dropout(sq.t().contiguous(), 0.5, (3, 3)))


def test_dropout_places_past_32_bits():
    """The groups' numbers pass 2^29, the byte offsets 2^32."""
    from wap_amd import ops
    n = (1 << 32) + 4096 + 5
    x = torch.ones(n, device=DEV, dtype=torch.bfloat16)
    y = ops.counter_dropout(x, 0.5, (11, 12), 3)
    assert y[:4096].max() == 2 and y[-4096:].max() == 2
    first = oracle.draws(64, 11, 12, 3) >= 32768
    assert torch.equal((y[:64] != 0).cpu(), first)
    at = (1 << 32) // 8
    low = 0xFFFFFFFF
    c, k = [at & low, (3 << 8) | (at >> 32), 12, 0], [11, 0]
    for _ in range(7):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(q >> 32) ^ c[1] ^ k[0], q & low, (p >> 32) ^ c[3] ^ k[1], p & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    want = torch.tensor([u for v in c for u in (v & 0xFFFF, v >> 16)]) >= 32768
    assert torch.equal((y[8 * at:8 * at + 8] != 0).cpu(), want)


# ------------------------------------------------------ streams, graphs, refusals

def test_on_another_stream():
    from wap_amd import ops
    g, h0, m, dh, dl = _scan_inputs(4, 900, 128, torch.bfloat16, 1, mask=True)
    logits, y, w, old, ref, adv = _loss_inputs(4, 30, 5000, torch.bfloat16, 1)

    def work():
        a = g.detach().requires_grad_()
        h, last = ops.gated_scan(a, h0, m)
        x = logits.detach().requires_grad_()
        l1, lp = ops.policy_loss(x, y, w, old, adv, ref, kl_coef=0.1)
        l2, mg = ops.preference_loss(x, y, w, ref)
        z = ops.counter_dropout(a, 0.2, (1, 1))
        return (h, last, l1, lp, l2, mg, z, *torch.autograd.grad((h, last), a, (dh, dl)),
                *torch.autograd.grad(l1, x), *torch.autograd.grad(l2, x))

    want = work()
    side = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(work())
    for s in side:
        torch.cuda.current_stream().wait_stream(s)
    for got in outs:
        assert all(torch.equal(a, c) for a, c in zip(want, got))


def test_captured_training_step_draws_anew_at_every_replay():
    """Forward and backward of the operators together in a graph, replayed
    with other inputs and another dropout step, against the eager result."""
    from wap_amd import ops
    torch.manual_seed(0)
    b, t, v, d = 4, 300, 130, 64
    p = {"emb": torch.randn(v, d), "w": torch.randn(d, 2 * d) * 0.3, "o": torch.randn(d, v) * 0.3}
    p = {n: x.to(DEV) for n, x in p.items()}
    x = torch.randint(v, (b, t), device=DEV)
    y = torch.randint(v, (b, t), device=DEV)
    mask = torch.ones(b, t, device=DEV)
    mask[1, 100:] = 0
    mask[3] = 0
    old = torch.full((b, t), -5.0, device=DEV)
    adv = torch.randn(b, device=DEV)
    rng = torch.tensor([5, 0], device=DEV)

    def step():
        q = {n: a.detach().requires_grad_() for n, a in p.items()}
        emb = q["emb"][x]
        h, _ = ops.gated_scan(emb @ q["w"], None, mask)
        h = ops.counter_dropout(h, 0.2, rng, 1, emb)
        logits = h @ q["o"]
        l1, _ = ops.policy_loss(logits, y, mask, old, adv, old, kl_coef=0.1)
        l2, _ = ops.preference_loss(logits, y, mask, old)
        s = ops.token_logprob(logits, y, mask).mean()
        total = l1 + l2 - s
        return [total.detach(), *torch.autograd.grad(total, (q["w"], q["o"]))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    drain()
    graphs = []
    for _ in range(2):  # two graphs of the same work, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, capture_error_mode="thread_local"):
            out = step()
        graphs.append((g, out))
    seen = []
    for i in range(6):
        rng[1] = i // 2
        y.copy_((y + i) % v)
        want = [w.clone() for w in step()]
        drain()
        g, out = graphs[i % 2]
        g.replay()
        drain()
        assert all(torch.equal(a, c) for a, c in zip(want, out)), i
        seen.append(float(out[0]))
    assert len(set(seen)) > 3


def test_captured_backward_alone_replays_to_the_same():
    """Forward and backward in two graphs; the backward one replayed again,
    with other upstream gradients, without the forward one."""
    from wap_amd import ops
    logits, y, w, old, ref, adv = _loss_inputs(3, 4, 500, torch.float32, 2)
    x = logits.requires_grad_()
    up = torch.ones((), device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss, _ = ops.policy_loss(x, y, w, old, adv, ref, kl_coef=0.1)
        want = torch.autograd.grad(loss, x)[0].clone()
        del loss
    torch.cuda.current_stream().wait_stream(side)
    drain()
    pool = torch.cuda.graph_pool_handle()
    fwd, bwd = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(fwd, pool=pool, capture_error_mode="thread_local"):
        loss, _ = ops.policy_loss(x, y, w, old, adv, ref, kl_coef=0.1)
    with torch.cuda.graph(bwd, pool=pool, capture_error_mode="thread_local"):
        d, = torch.autograd.grad(loss, x, up)
    fwd.replay()
    for s in (1.0, 4.0, 1.0, 0.5, 0.5, 0.0, 1.0):
        up.fill_(s)
        bwd.replay()
        drain()
        assert torch.equal(d, s * want), s
    fwd.replay()
    bwd.replay()
    drain()
    assert torch.equal(d, want)


def test_refused_on_the_gpu():
    from wap_amd import ops
    with pytest.raises(RuntimeError):
        ops.gated_scan(torch.zeros(2, 3, 4, dtype=torch.float64, device=DEV))
    with pytest.raises(ValueError):
        ops.gated_scan(torch.zeros(2, 3, 4, device=DEV), torch.zeros(2, 2))
    with pytest.raises(ValueError):
        ops.token_logprob(torch.zeros(2, 3, 4, device=DEV), torch.zeros(2, 3, dtype=torch.long))
    with pytest.raises(RuntimeError):
        ops.token_logprob(torch.zeros(2, 3, 4, dtype=torch.float64, device=DEV),
                          torch.zeros(2, 3, dtype=torch.long, device=DEV))
    with pytest.raises(ValueError):
        ops.counter_dropout(torch.zeros(4, device=DEV), 0.5, torch.zeros(2, dtype=torch.long))
    with pytest.raises(RuntimeError):
        ops.counter_dropout(torch.zeros(4, dtype=torch.float64, device=DEV), 0.5, (1, 1))


@pytest.mark.parametrize("b,t,d", [(0, 3, 4), (2, 0, 4), (2, 3, 0)])
def test_nothing_to_do(b, t, d):
    from wap_amd import ops
    h, last = ops.gated_scan(torch.zeros(b, t, 2 * d, device=DEV), torch.ones(b, d, device=DEV))
    assert h.shape == (b, t, d) and (last == 1).all() and last.shape == (b, d)
    assert ops.token_logprob(torch.zeros(0, 3, 4, device=DEV),
                             torch.zeros(0, 3, dtype=torch.long, device=DEV)).shape == (0, 3)
    assert ops.counter_dropout(torch.zeros(0, 5, device=DEV), 0.5, (1, 1)).shape == (0, 5)
