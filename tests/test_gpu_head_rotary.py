"""head_rotary and head_rotary_b against their formulas in 64 bits: both pair layouts, parts of the head, with
and without the norm and its weights, odd sizes, far positions, rows apart."""
import math

import pytest
import torch

from lmhelp import IDS, TYPES, U, apart, cuda, gen, normal, within

pytestmark = pytest.mark.gpu

EPS = 1e-6
# (tokens, heads of queries, of keys, head, rotated part)
SIZES = [(1, 1, 0, 2, 2), (3, 2, 1, 5, 4), (7, 3, 1, 8, 0), (5, 0, 2, 64, 64), (9, 4, 2, 80, 40), (300, 3, 1, 33, 18), (257, 8, 2, 128, 128), (70, 5, 5, 255, 254),
         (33, 2, 2, 256, 96), (2000, 4, 1, 96, 96)]


def _turn(x, angle, half):
    """The pairs of the last dimension turned by angle (t, 1, r / 2)."""
    c, s = torch.cos(angle), torch.sin(angle)
    a, b = x.chunk(2, -1) if half else (x[..., 0::2], x[..., 1::2])
    u, w = a * c - b * s, b * c + a * s
    return torch.cat([u, w], -1) if half else torch.stack([u, w], -1).flatten(-2)


def _pairs(x, half):
    """|a| + |b| of each value's pair."""
    a, b = (x.abs().chunk(2, -1)) if half else (x.abs()[..., 0::2], x.abs()[..., 1::2])
    return torch.cat([a + b, a + b], -1) if half else torch.stack([a + b, a + b], -1).flatten(-2)


def _inputs(size, dt, tg, far, seed=0):
    t, hq, hk, d, r = size
    g = gen(31 * t + d + seed)
    x = normal(g, t, (hq + hk) * d, dtype=dt)
    gq, gk = ((1 + 0.2 * torch.randn(d, generator=g)).to(tg) for _ in range(2))
    pos = torch.randint(-3, far, (t,), generator=g) if far else torch.arange(t)
    freq = 10000.0 ** (-torch.arange(r // 2, dtype=torch.float64) * 2 / max(r, 1))
    return x, gq, gk, pos, freq, normal(g, t, (hq + hk) * d, dtype=dt)


def _formula(size, x, gq, gk, pos, freq, half, norm, s):
    """(y, h, xh, rs, bound on y before its rounding) in 64 bits, heads apart."""
    t, hq, hk, d, r = size
    x = x.reshape(t, hq + hk, d)
    rs = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) if norm else torch.ones(t, hq + hk, 1, dtype=torch.float64)
    g = torch.cat([gq.expand(hq, d), gk.expand(hk, d)]) if norm else torch.ones(hq + hk, d, dtype=torch.float64)
    xh = x * rs
    h = xh * g
    angle = pos.double()[:, None, None] * freq
    y = torch.cat([s * _turn(h[..., :r], angle, half), h[..., r:]], -1)
    # rs: a sum nested at most 16 + 6 deep, a root, a division: 15 U; two products: 17 U of |h|.  The cosine is off by pi U
    # for the fraction of a turn, 3 U for the function and its factor, 2 U for the sum, and by three roundings in 64 bits of the
    # whole angle
    size_h = torch.cat([abs(s) * _pairs(h[..., :r], half), h[..., r:].abs()], -1)
    far = 2.0 ** -51 * float((pos.abs().max() * freq.max()) if freq.numel() and pos.numel() else 0)
    return y, h, xh, rs, g, (26 * U + far) * size_h, far


@pytest.mark.parametrize("half", [True, False], ids=["half", "neighbours"])
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "plain"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward(size, dt, norm, half):
    import stade_hip
    t, hq, hk, d, r = size
    tg = torch.float32 if d % 2 else dt
    x, gq, gk, pos, freq, _ = _inputs(size, dt, tg, 0 if t % 2 else 1000000)
    s = 1.0 if half else -0.75
    w = (gq, gk) if norm else (None, None)
    y = torch.full_like(x, 9.0).cuda()
    args = (*map(cuda, w), pos.cuda(), freq.cuda(), d, hq, hk, r, t)
    form = dict(norm=norm, eps=EPS, half=half, s=s)
    print(f"head_rotary {size} {IDS[dt]} norm={norm} half={half}", flush=True)
    stade_hip.head_rotary(y, x.cuda(), *args, **form)
    want, _, _, _, _, slack, _ = _formula(size, x.double(), gq.double(), gk.double(), pos, freq, half, norm, s)
    within("y", y, want.reshape(t, -1), slack.reshape(t, -1), dt)
    # rows apart, and in place: the same bits
    yv = apart(torch.zeros_like(y))
    stade_hip.head_rotary(yv, apart(x.cuda()), *args, **form)
    assert torch.equal(yv, y)
    stade_hip.head_rotary(yv, yv.copy_(x.cuda()), *args, **form)
    assert torch.equal(yv, y)


def _backward(size, yb, x, gq, gk, pos, freq, half, norm, s):
    t, hq, hk, d, r = size
    _, h, xh, rs, g, _, far = _formula(size, x, gq, gk, pos, freq, half, norm, s)
    yb = yb.reshape(t, hq + hk, d)
    hb = torch.cat([s * _turn(yb[..., :r], -pos.double()[:, None, None] * freq, half), yb[..., r:]], -1)
    eh = (9 * U + far) * torch.cat([abs(s) * _pairs(yb[..., :r], half), yb[..., r:].abs()], -1)
    if not norm:
        return hb, eh, None
    a = hb * g
    m = (a * xh).mean(-1, keepdim=True)
    # the mean: a sum nested at most 38 deep, a and xh off by eh |g| + U and 16 U
    em = (g.abs() * eh * xh.abs()).mean(-1, keepdim=True) + 60 * U * (a * xh).abs().mean(-1, keepdim=True)
    xb = rs * (a - xh * m)
    exb = rs * (g.abs() * eh + 18 * U * a.abs() + 35 * U * (xh * m).abs() + xh.abs() * em)
    sums = []
    for part in (slice(0, hq), slice(hq, hq + hk)):
        n = t * (part.stop - part.start)
        terms = (hb * xh)[:, part]
        sums.append((terms.sum((0, 1)), (n + 30) * U * terms.abs().sum((0, 1)) + (eh * xh.abs())[:, part].sum((0, 1))))
    return xb, exb, sums


@pytest.mark.parametrize("half", [True, False], ids=["half", "neighbours"])
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "plain"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_backward(size, dt, norm, half):
    import stade_hip
    t, hq, hk, d, r = size
    tg = torch.float32 if d % 2 else dt
    x, gq, gk, pos, freq, yb = _inputs(size, dt, tg, 0 if t % 2 else 1000000, seed=1)
    s = 1.0 if half else 1.5
    form = dict(norm=norm, eps=EPS, half=half, s=s)
    want, slack, sums = _backward(size, yb.double(), x.double(), gq.double(), gk.double(), pos, freq, half, norm, s)
    w = (gq.cuda(), gk.cuda()) if norm else (None, None)
    tail = (pos.cuda(), freq.cuda(), d, hq, hk, r, t)
    print(f"head_rotary_b {size} {IDS[dt]} norm={norm} half={half}", flush=True)
    for add in (False, True):
        g = gen(d)
        base, bq, bk = normal(g, t, (hq + hk) * d, dtype=dt), normal(g, d), normal(g, d)
        xb = base.cuda() if add else torch.full_like(base, float("nan")).cuda()
        gqb, gkb = ((v.cuda() if add else torch.full_like(v, float("nan")).cuda()) if norm else None for v in (bq, bk))
        stade_hip.head_rotary_b(yb.cuda(), x.cuda() if norm else None, xb, w[0], gqb, w[1], gkb, *tail, add=add, **form)
        to = want.reshape(t, -1) + (base.double() if add else 0)
        within("xb", xb, to, slack.reshape(t, -1) + 2 * U * to.abs(), dt)
        if norm:
            for got, b, (v, e) in ((gqb, bq, sums[0]), (gkb, bk, sums[1])):
                to = v + (b.double() if add else 0)
                within("weights", got, to, e + 2 * U * to.abs(), torch.float32)
    # rows apart: the same bits; only a part asked for: the same part
    xv, q2, k2 = apart(base.cuda()), bq.cuda(), bk.cuda()
    stade_hip.head_rotary_b(apart(yb.cuda()), apart(x.cuda()) if norm else None, xv, w[0], q2 if norm else None, w[1], None, *tail, add=True, **form)
    assert torch.equal(xv, xb) and (not norm or torch.equal(q2, gqb))
    if norm:
        stade_hip.head_rotary_b(yb.cuda(), x.cuda(), None, w[0], None, w[1], k2, *tail, add=True, **form)
        assert torch.equal(k2, gkb)


def test_far_positions():
    """Positions up to 2^31 turn by the angle's fraction: off by no more than near ones, and 2^-53 of the turns."""
    import stade_hip
    t, d = 64, 64
    x = normal(gen(3), t, d)
    pos = torch.randint(2 ** 30, 2 ** 31, (t,), generator=gen(4))
    freq = torch.from_numpy(stade_hip.rotary_freq(d))
    y = torch.empty(t, d, device="cuda")
    print("head_rotary far positions", flush=True)
    stade_hip.head_rotary(y, x.cuda(), None, None, pos.cuda(), freq.cuda(), d, 1, 0, d, t, norm=False)
    # (whole turns taken out of the angle in whole numbers: pos * freq by parts of 2^16)
    angle = ((pos >> 16).double()[:, None, None] * torch.remainder(freq * 65536.0, 2 * math.pi) + (pos & 65535).double()[:, None, None] * freq)
    want = _turn(x.double()[:, None], angle, True)[:, 0]
    within("y", y, want, (12 * U + 2.0 ** -53 * 2 ** 31 * 8) * _pairs(x.double(), True), torch.float32)


def test_no_tokens():
    import stade_hip
    e, i, f = torch.empty(0, 12, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), torch.ones(2, dtype=torch.float64, device="cuda")
    g, gb = torch.ones(4, device="cuda"), torch.ones(4, device="cuda")
    stade_hip.head_rotary(e, e, g, g, i, f, 4, 2, 1, 4, 0)
    stade_hip.head_rotary_b(e, e, e, g, gb, g, None, i, f, 4, 2, 1, 4, 0)
    assert gb.eq(1).all()
    stade_hip.head_rotary_b(e, e, e, g, gb, g, None, i, f, 4, 2, 1, 4, 0, add=False)
    assert not gb.any()


def test_values_that_are_not_finite():
    """A NaN or an infinity makes its own head NaN and no other."""
    import stade_hip
    t, h, d = 5, 4, 32
    x, pos, freq = normal(gen(1), t, h * d).cuda(), torch.arange(t).cuda(), torch.rand(d // 2, dtype=torch.float64).cuda()
    clean, y = torch.empty_like(x), torch.empty_like(x)
    stade_hip.head_rotary(clean, x, None, None, pos, freq, d, 3, 1, d, t)
    x[1, 2 * d + 3], x[4, 7] = float("inf"), float("nan")
    stade_hip.head_rotary(y, x, None, None, pos, freq, d, 3, 1, d, t)
    y, clean = y.view(t, h, d), clean.view(t, h, d)
    bad = torch.zeros(t, h, dtype=torch.bool, device="cuda")
    bad[1, 2] = bad[4, 0] = True
    assert torch.equal(torch.isnan(y).any(-1), bad) and torch.equal(y[~bad], clean[~bad])


def test_gradient_by_differences():
    """The directional derivative of <yb, head_rotary> by differences of the forward kernel."""
    import stade_hip
    size, h = (20, 2, 1, 24, 16), 2.0 ** -6
    t, hq, hk, d, r = size
    x, gq, gk, pos, freq, yb = (cuda(v) for v in _inputs(size, torch.float32, torch.float32, 0, seed=2))
    g = gen(9)
    dx, dq, dk = cuda(normal(g, t, (hq + hk) * d)), cuda(normal(g, d)), cuda(normal(g, d))

    def at(e):
        y = torch.empty_like(x)
        stade_hip.head_rotary(y, x + e * dx, gq + e * dq, gk + e * dk, pos, freq, d, hq, hk, r, t, eps=EPS)
        return (yb.double() * y.double()).sum()

    def exact(e):
        v = [(a.double() + e * b.double()).cpu() for a, b in ((x, dx), (gq, dq), (gk, dk))]
        return (yb.double().cpu().reshape(t, -1, d) * _formula(size, *v, pos.cpu(), freq.cpu(), True, True, 1.0)[0]).sum()

    xb, gqb, gkb = torch.zeros_like(x), torch.zeros_like(gq), torch.zeros_like(gk)
    stade_hip.head_rotary_b(yb, x, xb, gq, gqb, gk, gkb, pos, freq, d, hq, hk, r, t, eps=EPS)
    got = sum((a.double() * b.double()).sum() for a, b in ((xb, dx), (gqb, dq), (gkb, dk))).cpu()
    numeric, curved = ((at(h) - at(-h)) / (2 * h)).cpu(), abs((exact(h) - exact(-h)) / (2 * h) - got)
    # y is off by 26 U of a pair (above), its inputs by 2 U of themselves: 30 U of some 4 |yb| each, at two points
    assert abs(numeric - got) <= curved + 2 * 30 * U * 4 * yb.double().abs().sum().cpu() / (2 * h)
    wxb, sxb, sums = _backward(size, *(v.double().cpu() for v in (yb, x, gq, gk)), pos.cpu(), freq.cpu(), True, True, 1.0)
    want = (wxb.reshape(t, -1) * dx.double().cpu()).sum() + sum((v * b.double().cpu()).sum() for (v, _), b in zip(sums, (dq, dk)))
    bound = (sxb.reshape(t, -1) * dx.double().cpu().abs()).sum() + sum((e * b.double().cpu().abs()).sum() for (_, e), b in zip(sums, (dq, dk)))
    assert abs(got - want) <= bound + 8 * U * abs(want) + U * (xb.abs() * dx.abs()).sum().cpu()


def test_frequencies():
    """By the formula: all pairs, and by parts of the trained context."""
    import numpy as np
    import stade_hip
    j = np.arange(32)
    f = 500000.0 ** (-2 * j / 64)
    assert np.allclose(stade_hip.rotary_freq(64, 500000.0), f, rtol=1e-14)
    assert np.allclose(stade_hip.rotary_freq(64, 500000.0, factor=4.0), f / 4, rtol=1e-14)
    got = stade_hip.rotary_freq(64, 500000.0, factor=8.0, length=8192.0, low=1.0, high=4.0)
    turns = 8192.0 * f / (2 * np.pi)
    keep = np.clip((turns - 1) / 3, 0, 1)
    assert np.allclose(got, f * (keep + (1 - keep) / 8), rtol=1e-13)
    assert (got[turns >= 4] == stade_hip.rotary_freq(64, 500000.0)[turns >= 4]).all() and (turns < 1).any() and (turns > 4).any()
    assert stade_hip.rotary_freq(0).size == 0
