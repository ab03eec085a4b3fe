"""layernorm and layernorm_b against their formulas in 64 bits, from x and from its 8-bit tape."""
import pytest
import torch

from lmhelp import IDS, TYPES, U, apart, cuda, gen, new_tape, normal, tape_values, within

pytestmark = pytest.mark.gpu

# the lengths on both sides of each step of the kernels' forms, and rows that are read again
SIZES = [(1, 1), (3, 2), (5, 127), (9, 128), (4, 129), (7, 512), (6, 513), (2, 1025), (3, 2049), (5, 4100), (2, 8200), (3, 16385),
         (2, 32769), (2, 70003), (700, 96), (1300, 257), (2500, 1030)]
EPS = 1e-5
# how deep the sums of a row nest: at most 72 values a thread up to 70003 columns in the long form,
# some 64 in the others; then 6 steps over a wave and 16 over the waves
DEPTH = 100


def _inputs(n, d, dt, tg, seed=0):
    g = gen(n * 31 + d + seed)
    x = (torch.randn(n, d, generator=g) * torch.exp(torch.randn(n, 1, generator=g)) + 0.5).to(dt)
    return x, (1 + 0.2 * torch.randn(d, generator=g)).to(tg), (0.3 * torch.randn(d, generator=g)).to(tg), normal(g, n, d, dtype=dt)


def _stats(x):
    mu = x.mean(1, keepdim=True)
    return mu, 1.0 / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + EPS)


def _forward(x, g, b):
    """(y, mu, rs) of x in 64 bits, and the bound on y's error before its rounding."""
    mu, rs = _stats(x)
    xh = (x - mu) * rs
    y = xh * g + b
    dmu = DEPTH * U * x.abs().mean(1, keepdim=True)
    # x - mu moves by dmu and its own rounding; rs by half the variance's error, the error of the
    # mean squared, and a few roundings
    rel = DEPTH * U + (dmu * rs) ** 2
    return y, mu, rs, g.abs() * (rs * dmu + xh.abs() * (rel + 4 * U)) + 2 * U * (y.abs() + b.abs()), dmu, rel


@pytest.mark.parametrize("tape", [False, True], ids=["x", "tape"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward(size, dt, tape):
    import stade_hip
    n, d = size
    tg = torch.float32 if d % 2 else dt
    x, g, b, _ = _inputs(n, d, dt, tg)
    print(f"layernorm n={n} d={d} {IDS[dt]} tape={tape}", flush=True)
    y = torch.full((n, d), 9.0, dtype=dt, device="cuda")
    mu, rs = (torch.empty(n, device="cuda") for _ in range(2))
    t = new_tape(d, n) if tape else None
    stade_hip.layernorm(y, x.cuda(), g.cuda(), b.cuda(), mu, rs, d, n, eps=EPS, tape=t)
    wy, wmu, wrs, slack, dmu, rel = _forward(x.double(), g.double(), b.double())
    within("y", y, wy, slack, dt)
    within("mu", mu, wmu[:, 0], dmu[:, 0], torch.float32)
    within("rs", rs, wrs[:, 0], (rel * wrs)[:, 0] + 4 * U * wrs[:, 0], torch.float32)
    if tape:
        back = torch.empty(n, d, dtype=dt, device="cuda")
        stade_hip.tape8_load(*t, back, d, n)
        assert torch.equal(back.double().cpu(), tape_values(x.double()))
    yv = apart(torch.zeros(n, d, dtype=dt, device="cuda"))
    stade_hip.layernorm(yv, apart(x.cuda()), g.cuda(), b.cuda(), None, None, d, n, eps=EPS)
    assert torch.equal(yv, y)


def _backward(yb, x, g, mu, rs):
    """(xb, gb, bb) in 64 bits and their bounds."""
    xh = (x - mu) * rs
    a = yb * g
    m0, m1 = a.mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
    xb = rs * (a - m0 - xh * m1)
    # xh is off by 3 roundings of (|x| + |mu|) rs
    dxh = 3 * U * (x.abs() + mu.abs()) * rs
    d0 = DEPTH * U * a.abs().mean(1, keepdim=True)
    d1 = DEPTH * U * (a * xh).abs().mean(1, keepdim=True) + (a.abs() * dxh).mean(1, keepdim=True)
    sxb = rs * (4 * U * (a.abs() + m0.abs() + (xh * m1).abs()) + d0 + xh.abs() * d1 + dxh * m1.abs()) + 2 * U * xb.abs()
    n = x.shape[0]   # the rows' sums nest at most n deep
    sgb = (n + 4) * U * (yb * xh).abs().sum(0) + (yb.abs() * dxh).sum(0)
    sbb = (n + 4) * U * yb.abs().sum(0)
    return xb, (yb * xh).sum(0), yb.sum(0), sxb, sgb, sbb


@pytest.mark.parametrize("add", [False, True], ids=["set", "add"])
@pytest.mark.parametrize("tape", [False, True], ids=["x", "tape"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_backward(size, dt, tape, add):
    import stade_hip
    n, d = size
    tg = torch.float32 if d % 2 else dt
    x, g, _, yb = _inputs(n, d, dt, tg, seed=1)
    r = gen(n + 3 * d)
    base = [normal(r, n, d, dtype=dt), normal(r, d), normal(r, d)]
    mu, rs = (v.float() for v in _stats(x.double()))
    print(f"layernorm_b n={n} d={d} {IDS[dt]} tape={tape} add={add}", flush=True)
    t = None
    if tape:
        t = new_tape(d, n)
        stade_hip.tape8_store(x.cuda(), *t, d, n)
    held = tape_values(x.double()) if tape else x.double()
    wxb, wgb, wbb, sxb, sgb, sbb = _backward(yb.double(), held, g.double(), mu.double(), rs.double())
    if add:
        wxb, wgb, wbb = (w + v.double() for w, v in zip((wxb, wgb, wbb), base))

    def go(xb, yb, x):
        gb, bb = (base[k].cuda() if add else torch.full((d,), float("nan"), device="cuda") for k in (1, 2))
        stade_hip.layernorm_b(yb, None if tape else x, xb, g.cuda(), gb, bb, mu[:, 0].cuda(), rs[:, 0].cuda(), d, n, add=add, tape=t)
        return gb, bb

    xb = base[0].cuda() if add else torch.full((n, d), float("nan"), dtype=dt, device="cuda")
    gb, bb = go(xb, yb.cuda(), x.cuda())
    within("xb", xb, wxb, sxb + 2 * U * wxb.abs(), dt)
    within("gb", gb, wgb, sgb, torch.float32)
    within("bb", bb, wbb, sbb, torch.float32)
    # rows apart: the same bits
    xv = apart(base[0].cuda())
    gv, bv = go(xv, apart(yb.cuda()), apart(x.cuda()))
    assert torch.equal(xv, xb) and torch.equal(gv, gb) and torch.equal(bv, bb)


def test_parts_left_out():
    """No weights; no shadow of the weights; no shadow of the rows; and xb in yb's place."""
    import stade_hip
    n, d = 37, 300
    x, g, _, yb = (cuda(v) for v in _inputs(n, d, torch.float32, torch.float32))
    mu, rs = (v.float() for v in _stats(x.double()))
    y = torch.empty(n, d, device="cuda")
    stade_hip.layernorm(y, x, None, None, None, None, d, n, eps=EPS)
    one, none = torch.ones(d, dtype=torch.float64, device="cuda"), torch.zeros(d, dtype=torch.float64, device="cuda")
    wy, _, _, slack, _, _ = _forward(x.double(), one, none)
    within("y", y, wy, slack, torch.float32)
    wxb, wgb, wbb, sxb, sgb, sbb = _backward(yb.double(), x.double(), one, mu.double(), rs.double())
    xb = torch.empty(n, d, device="cuda")
    stade_hip.layernorm_b(yb, x, xb, None, None, None, mu[:, 0].contiguous(), rs[:, 0].contiguous(), d, n, add=False)
    within("xb", xb, wxb, sxb, torch.float32)
    gb, bb = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    stade_hip.layernorm_b(yb, x, None, None, gb, bb, mu[:, 0].contiguous(), rs[:, 0].contiguous(), d, n, add=False)
    within("gb", gb, wgb, sgb, torch.float32)
    within("bb", bb, wbb, sbb, torch.float32)
    only = torch.empty(d, device="cuda")
    stade_hip.layernorm_b(yb, x, None, None, None, only, mu[:, 0].contiguous(), rs[:, 0].contiguous(), d, n, add=False)
    assert torch.equal(only, bb)
    same = yb.clone()
    stade_hip.layernorm_b(same, x, same, None, None, None, mu[:, 0].contiguous(), rs[:, 0].contiguous(), d, n, add=False)
    assert torch.equal(same, xb)


@pytest.mark.parametrize("d", [100, 640])
def test_tape_of_the_largest_values(d):
    """Scales at the top of the exponent range, where 128 of their units are infinite."""
    import stade_hip
    n = 5
    x, g, _, yb = _inputs(n, d, torch.float32, torch.float32, seed=4)
    x = (x.double().clamp(-3, 3) * 2.0 ** 124).float()
    mu, rs = torch.zeros(n), torch.full((n,), 2.0 ** -124)
    t = new_tape(d, n)
    stade_hip.tape8_store(x.cuda(), *t, d, n)
    xb = torch.empty(n, d, device="cuda")
    gb, bb = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    stade_hip.layernorm_b(yb.cuda(), None, xb, g.cuda(), gb, bb, mu.cuda(), rs.cuda(), d, n, add=False, tape=t)
    # (rs scales xb into subnormals, which are rounded to their own least)
    wxb, wgb, wbb, sxb, sgb, sbb = _backward(yb.double(), tape_values(x.double()), g.double(), mu.double()[:, None], rs.double()[:, None])
    within("gb", gb, wgb, sgb, torch.float32)
    within("bb", bb, wbb, sbb, torch.float32)
    within("xb", xb, wxb, sxb + 2.0 ** -126, torch.float32)


def test_no_rows():
    import stade_hip
    e, d = torch.empty(0, 6, device="cuda"), 6
    n = torch.empty(0, device="cuda")
    gb, bb = torch.ones(d, device="cuda"), torch.ones(d, device="cuda")
    stade_hip.layernorm(e, e, None, None, n, n, d, 0)
    stade_hip.layernorm_b(e, e, e, None, gb, bb, n, n, d, 0)
    assert gb.eq(1).all() and bb.eq(1).all()
    stade_hip.layernorm_b(e, e, e, None, gb, bb, n, n, d, 0, add=False)
    assert not gb.any() and not bb.any()


def test_values_that_are_not_finite():
    """An infinity or a NaN makes its own row NaN and no other."""
    import stade_hip
    n, d = 6, 200
    x, g, b, _ = (cuda(v) for v in _inputs(n, d, torch.float32, torch.float32))
    clean = torch.empty(n, d, device="cuda")
    stade_hip.layernorm(clean, x, g, b, None, None, d, n)
    x[1, 3], x[4, 199] = float("inf"), float("nan")
    y = torch.empty(n, d, device="cuda")
    stade_hip.layernorm(y, x, g, b, None, None, d, n)
    bad = torch.tensor([1, 4], device="cuda")
    ok = torch.tensor([0, 2, 3, 5], device="cuda")
    assert torch.isnan(y[bad]).all() and torch.equal(y[ok], clean[ok])


def test_gradient_by_differences():
    """The directional derivative of <yb, layernorm> by differences of the forward kernel."""
    import stade_hip
    n, d, h = 20, 130, 2.0 ** -6
    x, g, b, yb = (cuda(v) for v in _inputs(n, d, torch.float32, torch.float32, seed=5))
    r = gen(8)
    dx, dg, db = cuda(normal(r, n, d)), cuda(normal(r, d)), cuda(normal(r, d))

    def at(s, kernel):
        xs, gs, bs = x + s * dx, g + s * dg, b + s * db
        if not kernel:
            return (yb.double() * _forward(x.double() + s * dx.double(), g.double() + s * dg.double(), b.double() + s * db.double())[0]).sum()
        y = torch.empty(n, d, device="cuda")
        stade_hip.layernorm(y, xs, gs, bs, None, None, d, n, eps=EPS)
        return (yb.double() * y.double()).sum()

    mu, rs = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    y, xb = torch.empty(n, d, device="cuda"), torch.zeros(n, d, device="cuda")
    gb, bb = torch.zeros(d, device="cuda"), torch.zeros(d, device="cuda")
    stade_hip.layernorm(y, x, g, b, mu, rs, d, n, eps=EPS)
    stade_hip.layernorm_b(yb, x, xb, g, gb, bb, mu, rs, d, n)
    got = sum((p.double() * q.double()).sum() for p, q in ((xb, dx), (gb, dg), (bb, db)))
    numeric = (at(h, True) - at(-h, True)) / (2 * h)
    # the differences' own error: what they are off by in 64 bits, and the kernel's and the inputs'
    # rounding (an input's moves y by at most rs |g| per unit, twice over for the means) over h
    wxb, wgb, wbb, sxb, sgb, sbb = _backward(yb.double(), x.double(), g.double(), *(v.double()[:, None] for v in (mu, rs)))
    exact = sum((p * q.double()).sum() for p, q in ((wxb, dx), (wgb, dg), (wbb, db)))
    curved = abs((at(h, False) - at(-h, False)) / (2 * h) - exact)
    _, _, wrs, slack, _, _ = _forward(x.double(), g.double(), b.double())
    moved = slack + 3 * U * x.double().abs() * wrs * g.double().abs() + U * (g.double().abs() * 5 + b.double().abs())
    formula = (sxb * dx.double().abs()).sum() + (sgb * dg.double().abs()).sum() + (sbb * db.double().abs()).sum()
    assert abs(got - exact) <= formula
    assert abs(numeric - got) <= curved + (yb.double().abs() * moved).sum() * 2 / h + formula
