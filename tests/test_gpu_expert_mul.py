"""expert_mul and expert_mul_b against products in 64 bits, expert by expert."""
import pytest
import torch

from lmhelp import IDS, TYPES, U, apart, cuda, gen, new_tape, normal, tape_values, within

pytestmark = pytest.mark.gpu

# (rows of each expert, rows of none after them, i_in, i_out)
SIZES = [([1], 0, 1, 1), ([0, 1, 0], 0, 5, 3), ([3, 0, 7], 2, 33, 40), ([64, 65, 1], 0, 64, 64), ([17] * 70, 0, 40, 24),
         ([130, 0, 257], 5, 96, 200), ([300, 1, 0, 100], 0, 515, 130), ([128, 256], 0, 256, 256), ([0, 0], 9, 16, 8), ([5, 900], 0, 130, 700),
         ([32, 0, 16], 0, 1000, 512), ([0, 600], 0, 264, 1032)]
NAME = lambda s: f"{len(s[0])}x{sum(s[0])}+{s[1]}-{s[2]}-{s[3]}"   # noqa: E731


def _case(size, dt, seed=0):
    counts, rest, i, o = size
    t, e = sum(counts) + rest, len(counts)
    g = gen(t * 13 + i + o + seed)
    start = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(torch.tensor(counts), 0)])
    return t, e, i, o, start, normal(g, t, i, dtype=dt), normal(g, e, i, o, dtype=dt, scale=i ** -0.5), normal(g, t, o, dtype=dt), g


def _y(x, w, start):
    y, size = torch.zeros(x.shape[0], w.shape[2], dtype=torch.float64), torch.zeros(x.shape[0], w.shape[2], dtype=torch.float64)
    for e in range(w.shape[0]):
        r = slice(int(start[e]), int(start[e + 1]))
        y[r], size[r] = x[r] @ w[e], x[r].abs() @ w[e].abs()
    return y, size


def _wb(x, yb, start, e):
    out = torch.zeros(2, e, x.shape[1], yb.shape[1], dtype=torch.float64)
    for k in range(e):
        r = slice(int(start[k]), int(start[k + 1]))
        out[0, k], out[1, k] = x[r].t() @ yb[r], x[r].t().abs() @ yb[r].abs()
    return out


@pytest.mark.parametrize("add", [False, True], ids=["set", "add"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", SIZES, ids=NAME)
def test_forward(size, dt, add):
    import stade_hip
    t, e, i, o, start, x, w, _, g = _case(size, dt)
    base = normal(g, t, o, dtype=dt)
    print(f"expert_mul {NAME(size)} {IDS[dt]} add={add}", flush=True)
    y = base.cuda() if add else torch.full((t, o), float("nan"), dtype=dt, device="cuda")
    stade_hip.expert_mul(y, x.cuda(), w.cuda(), start.cuda(), i, o, t, e, add=add, check=True)
    want, scale = _y(x.double(), w.double(), start)
    if add:
        want = want + base.double()
    # products of 16-bit values are exact in fp32; sums nest at most i deep
    within("y", y, want, U * ((i + 4) * scale + 2 * want.abs()), dt)
    yv = apart(base.cuda())
    stade_hip.expert_mul(yv, apart(x.cuda()), w.cuda(), start.cuda(), i, o, t, e, add=add)
    assert torch.equal(yv, y)


@pytest.mark.parametrize("add", [False, True], ids=["set", "add"])
@pytest.mark.parametrize("held", ["x", "tape"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", SIZES, ids=NAME)
def test_backward(size, dt, held, add):
    import stade_hip
    t, e, i, o, start, x, w, yb, g = _case(size, dt, seed=1)
    twb = dt if o % 3 == 0 else torch.float32
    bx, bw = normal(g, t, i, dtype=dt), normal(g, e, i, o, dtype=twb)
    print(f"expert_mul_b {NAME(size)} {IDS[dt]} {held} add={add}", flush=True)
    tape, kept = None, x.double()
    if held == "tape":
        tape = new_tape(i, t)
        stade_hip.tape8_store(x.cuda(), *tape, i, t)
        kept = tape_values(x.double())

    def go(xb, yb, x):
        wb = bw.cuda() if add else torch.full((e, i, o), float("nan"), dtype=twb, device="cuda")
        stade_hip.expert_mul_b(yb, None if tape else x, xb, w.cuda(), wb, start.cuda(), i, o, t, e, add=add, tape=tape, check=True)
        return wb

    xb = bx.cuda() if add else torch.full((t, i), float("nan"), dtype=dt, device="cuda")
    wb = go(xb, yb.cuda(), x.cuda())
    wxb, sxb = _y(yb.double(), w.double().transpose(1, 2), start)
    wwb, swb = _wb(kept, yb.double(), start, e)
    if add:
        wxb, wwb = wxb + bx.double(), wwb + bw.double()
    within("xb", xb, wxb, U * ((o + 4) * sxb + 2 * wxb.abs()), dt)
    longest = max(size[0])
    within("wb", wb, wwb, U * ((longest + 8) * swb + 2 * wwb.abs()), twb)
    xv = apart(bx.cuda())
    wv = go(xv, apart(yb.cuda()), apart(x.cuda()))
    assert torch.equal(xv, xb) and torch.equal(wv, wb)
    # one shadow at a time
    x1 = bx.cuda() if add else torch.empty(t, i, dtype=dt, device="cuda")
    stade_hip.expert_mul_b(yb.cuda(), None, x1, w.cuda(), None, start.cuda(), i, o, t, e, add=add)
    assert torch.equal(x1, xb)
    w1 = bw.cuda() if add else torch.empty(e, i, o, dtype=twb, device="cuda")
    stade_hip.expert_mul_b(yb.cuda(), None if tape else x.cuda(), None, None, w1, start.cuda(), i, o, t, e, add=add, tape=tape)
    assert torch.equal(w1, wb)


def test_rows_of_no_expert_on_both_sides():
    """Rows before start[0] and from start[i_e] on have no expert, also where they hold NaN."""
    import stade_hip
    t, e, i, o = 100, 2, 64, 72
    g = gen(4)
    x, w, yb = normal(g, t, i), normal(g, e, i, o), normal(g, t, o)
    x[:7], x[90:], yb[:7], yb[90:] = (float("nan"),) * 4
    start = torch.tensor([7, 50, 90])
    y, xb = torch.full((t, o), 3.0, device="cuda"), torch.full((t, i), 3.0, device="cuda")
    wb = torch.empty(e, i, o, device="cuda")
    stade_hip.expert_mul(y, x.cuda(), w.cuda(), start.cuda(), i, o, t, e)
    stade_hip.expert_mul_b(yb.cuda(), x.cuda(), xb, w.cuda(), wb, start.cuda(), i, o, t, e, add=False)
    for v in (y, xb):
        assert not v[:7].any() and not v[90:].any()
    xs, ys = x.double(), yb.double()
    want, scale = _y(xs[7:90], w.double(), start - 7)
    within("y", y[7:90], want, U * (i + 4) * scale, torch.float32)
    wwb, swb = _wb(xs[7:90], ys[7:90], start - 7, e)
    within("wb", wb, wwb, U * 60 * swb, torch.float32)


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
def test_values_that_are_not_finite_stay_in_their_rows(dt):
    import stade_hip
    counts, i, o = [70, 3, 60], 96, 80
    t, e, i, o, start, x, w, yb, _ = _case((counts, 0, i, o), dt)
    y0 = torch.empty(t, o, dtype=dt, device="cuda")
    stade_hip.expert_mul(y0, x.cuda(), w.cuda(), start.cuda(), i, o, t, e)
    x[69, 0], x[73, 95] = float("nan"), float("inf")
    y = torch.empty(t, o, dtype=dt, device="cuda")
    stade_hip.expert_mul(y, x.cuda(), w.cuda(), start.cuda(), i, o, t, e)
    hit = torch.zeros(t, dtype=torch.bool)
    hit[69] = hit[73] = True
    assert torch.equal(y.cpu()[~hit], y0.cpu()[~hit])
    assert torch.isnan(y[69]).all() and not torch.isfinite(y[73]).any()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=IDS.get)
def test_tape_of_the_largest_values(dt):
    """Scales at the top of the exponent range, where 128 of their units are infinite."""
    import stade_hip
    t, e, i, o, start, x, _, yb, _ = _case(([70, 20], 0, 64, 72), dt, seed=3)
    x, yb = (x.double() * 2.0 ** 124).to(dt), (yb.double() * 2.0 ** -120).to(dt)
    tape = new_tape(i, t)
    stade_hip.tape8_store(x.cuda(), *tape, i, t)
    wb = torch.empty(e, i, o, device="cuda")
    stade_hip.expert_mul_b(yb.cuda(), None, None, None, wb, start.cuda(), i, o, t, e, add=False, tape=tape)
    want, scale = _wb(tape_values(x.double()), yb.double(), start, e)
    within("wb", wb, want, U * 78 * scale, torch.float32)


def test_offsets_that_are_wrong_raise_the_flag():
    import stade_hip
    t, e, i, o = 64, 3, 32, 32
    g = gen(2)
    x, w, y = cuda(normal(g, t, i)), cuda(normal(g, e, i, o)), torch.empty(t, o, device="cuda")
    xb, wb = torch.empty(t, i, device="cuda"), torch.empty(e, i, o, device="cuda")
    for bad in ([0, 40, 20, 64], [0, 10, 20, 999], [-5, 10, 20, 64]):
        print(f"expert_mul start={bad}", flush=True)
        start = torch.tensor(bad, device="cuda")
        with pytest.raises(stade_hip.StadeHipBoundsError):
            stade_hip.expert_mul(y, x, w, start, i, o, t, e, check=True)
        with pytest.raises(stade_hip.StadeHipBoundsError):
            stade_hip.expert_mul_b(y, x, xb, w, wb, start, i, o, t, e, add=False, check=True)
    assert stade_hip.device_error() == 0


def test_decreasing_offsets_raise_the_flag_of_wb_alone():
    import stade_hip
    g = gen(2)
    for e in (3, 70):
        x, yb, wb = cuda(normal(g, 64, 32)), cuda(normal(g, 64, 32)), torch.empty(e, 32, 32, device="cuda")
        for at in (2, e):
            print(f"expert_mul_b wb alone, experts {e}, decreasing at {at}", flush=True)
            start = torch.full((e + 1,), 40)
            start[0], start[at] = 0, 20
            with pytest.raises(stade_hip.StadeHipBoundsError):
                stade_hip.expert_mul_b(yb, x, None, None, wb, start.cuda(), 32, 32, 64, e, add=False, check=True)
    assert stade_hip.device_error() == 0


def test_nothing():
    import stade_hip
    start = torch.zeros(4, dtype=torch.int64, device="cuda")
    e = torch.empty(0, 8, device="cuda")
    w, wb = torch.randn(3, 8, 8, device="cuda"), torch.ones(3, 8, 8, device="cuda")
    stade_hip.expert_mul(e, e, w, start, 8, 8, 0, 3)
    stade_hip.expert_mul_b(e, e, e, w, wb, start, 8, 8, 0, 3)
    assert wb.eq(1).all()
    stade_hip.expert_mul_b(e, e, e, w, wb, start, 8, 8, 0, 3, add=False)
    assert not wb.any()
    # no input columns: products of nothing
    y = torch.ones(5, 8, device="cuda")
    start[1:] = 5
    stade_hip.expert_mul(y, torch.empty(5, 0, device="cuda"), torch.empty(0, device="cuda"), start, 0, 8, 5, 3)
    assert not y.any()
    # no output columns: a shadow of nothing
    xb = torch.ones(5, 8, device="cuda")
    stade_hip.expert_mul_b(torch.empty(5, 0, device="cuda"), None, xb, None, None, start, 8, 0, 5, 3, add=False)
    assert not xb.any()
    # no experts
    stade_hip.expert_mul(y.fill_(1), torch.randn(5, 8, device="cuda"), None or torch.empty(0, device="cuda"), start[:1], 8, 8, 5, 0)
    assert not y.any()


def test_gradient_by_differences():
    """Bilinear: <yb, f(x + dx, w) - f(x - dx, w)> / 2 = <xb, dx>, and the same for w."""
    import stade_hip
    t, e, i, o, start, x, w, yb, g = _case(([40, 0, 77], 0, 60, 50), torch.float32)
    dx, dw = normal(g, t, i), normal(g, e, i, o)
    c = lambda v: v.cuda()   # noqa: E731
    xb, wb = torch.zeros(t, i, device="cuda"), torch.zeros(e, i, o, device="cuda")
    stade_hip.expert_mul_b(c(yb), c(x), xb, c(w), wb, c(start), i, o, t, e)

    def f(x, w):
        y = torch.empty(t, o, device="cuda")
        stade_hip.expert_mul(y, c(x), c(w), c(start), i, o, t, e)
        return y.double()

    ybd = c(yb).double()
    size = lambda a, b: _y(a.double().abs(), b.double().abs(), start)[0].cuda()   # noqa: E731
    for got, want, bound in (((f(x + dx, w) - f(x - dx, w)) / 2, (xb.double() * c(dx).double()).sum(), size(x.abs() + dx.abs(), w)),
                             ((f(x, w + dw) - f(x, w - dw)) / 2, (wb.double() * c(dw).double()).sum(), size(x, w.abs() + dw.abs()))):
        # sums nest at most 80 deep on either side, and the shifted inputs are rounded once
        assert abs((ybd * got).sum() - want) <= 2 * 90 * U * (ybd.abs() * bound).sum()


# few tiles and a long k: of y, of xb and of wb; whole and aligned, and odd
LONG = [([20, 0, 30], 3, 2000, 72), ([40], 1, 64, 2104), ([1500, 700], 2, 56, 64), ([20, 0, 30], 3, 2001, 71), ([40], 1, 65, 2103),
        ([1500, 700], 2, 51, 67)]


@pytest.mark.parametrize("add", [False, True], ids=["set", "add"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", LONG, ids=NAME)
def test_long_k(size, dt, add):
    test_forward(size, dt, add)
    test_backward(size, dt, "x", add)
    test_backward(size, dt, "tape", add)


# sizes that make a round of the largest tiles and more (256 x 256 on 256 CUs): of y, of xb and of wb; whole
# and aligned, and odd
LARGE = [([700, 300, 513], 3, 64, 16384), ([700, 513], 0, 16384, 72), ([70, 0, 33], 0, 4104, 4096), ([700, 300, 513], 0, 67, 16389),
         ([1213], 5, 16389, 35), ([70, 33], 0, 4099, 4103)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=IDS.get)
@pytest.mark.parametrize("size", LARGE, ids=NAME)
def test_large_tiles(size, dt):
    import stade_hip
    t, e, i, o, start, x, w, yb, g = _case(size, dt, seed=2)
    print(f"expert_mul large {NAME(size)} {IDS[dt]}", flush=True)
    xc, wc, ybc, sc = x.cuda(), w.cuda(), yb.cuda(), start.cuda()
    y = torch.full((t, o), float("nan"), dtype=dt, device="cuda")
    stade_hip.expert_mul(y, xc, wc, sc, i, o, t, e)
    want, scale = _y(x.double(), w.double(), start)
    within("y", y, want, U * (i + 4) * scale, dt)
    xb = torch.full((t, i), float("nan"), dtype=dt, device="cuda")
    wb = torch.full((e, i, o), float("nan"), device="cuda")
    stade_hip.expert_mul_b(ybc, xc, xb, wc, wb, sc, i, o, t, e, add=False)
    want, scale = _y(yb.double(), w.double().transpose(1, 2), start)
    within("xb", xb, want, U * (o + 4) * scale, dt)
    want, scale = _wb(x.double(), yb.double(), start, e)
    within("wb", wb, want, U * (max(size[0]) + 8) * scale, torch.float32)
    # from the tape, added to what is there
    tape = new_tape(i, t)
    stade_hip.tape8_store(xc, *tape, i, t)
    base = wb.double().cpu()
    stade_hip.expert_mul_b(ybc, None, None, None, wb, sc, i, o, t, e, tape=tape)
    want, scale = _wb(tape_values(x.double()), yb.double(), start, e)
    within("wb from the tape", wb, base + want, U * ((max(size[0]) + 8) * scale + 2 * (base + want).abs()), torch.float32)
