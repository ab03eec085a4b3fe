"""attention and attention_b against their formulas in 64 bits: ragged sequences, groups of heads, windows and sinks,
lengths at the tiles' ends, rows that see nothing, odd heads, rows apart."""
import pytest
import torch

from attnhelp import Case, formula
from lmhelp import IDS, TYPES, U, apart, gen, normal, within

pytestmark = pytest.mark.gpu

F, B, H = torch.float32, torch.bfloat16, torch.float16
# sequences (queries, keys), heads of queries and keys, head, window, sinks, columns of none before and behind
CASES = {
    "one key": ([(1, 1)], 1, 1, 8, None, 0, 0, 0),
    "one query": ([(1, 70)], 4, 2, 64, None, 0, 0, 0),
    "tile ends": ([(31, 31), (32, 32), (33, 33), (63, 64), (64, 65), (65, 65)], 1, 1, 64, None, 0, 0, 0),
    "block ends": ([(127, 127), (128, 128), (129, 130)], 2, 1, 32, None, 0, 0, 0),
    "window": ([(300, 300), (129, 129)], 2, 2, 128, 50, 0, 0, 0),
    "window of one": ([(70, 70)], 2, 1, 40, 1, 0, 0, 0),
    "window and sinks": ([(400, 400), (5, 5), (260, 300)], 4, 1, 128, 70, 4, 0, 0),
    "sinks past a tile": ([(300, 300)], 3, 1, 64, 33, 40, 0, 0),
    "most sinks": ([(500, 500)], 2, 2, 24, 20, 64, 0, 0),
    "sinks alone": ([(200, 200)], 2, 1, 16, 0, 3, 0, 0),
    "nothing seen": ([(60, 60)], 2, 1, 16, 0, 0, 0, 0),
    "more queries than keys": ([(40, 7), (3, 0), (150, 20)], 2, 1, 64, None, 0, 0, 0),
    "empty ones": ([(0, 0), (5, 5), (0, 9), (0, 0), (20, 33), (0, 0)], 2, 2, 64, None, 0, 0, 0),
    "columns of none": ([(33, 40), (2, 100)], 4, 2, 64, 30, 2, 5, 150),
    "only columns of none": ([(0, 0)], 2, 1, 32, None, 0, 0, 140),
    "chunk of a long one": ([(30, 900), (1, 700)], 6, 2, 128, None, 0, 0, 0),
    "single tokens": ([(1, k) for k in (1, 2, 31, 32, 33, 64, 127, 128, 129, 500, 1000, 7)], 8, 2, 128, None, 0, 0, 0),
    "single tokens, window": ([(1, k) for k in (1, 40, 41, 300, 1000)], 5, 1, 80, 40, 3, 0, 0),
    "groups of 3": ([(150, 150), (77, 99)], 6, 2, 64, 40, 2, 0, 0),
    "groups of 12": ([(45, 45)], 12, 1, 32, None, 0, 0, 0),
    "groups of 40": ([(9, 30), (20, 20)], 40, 1, 32, 11, 1, 0, 0),
    "group wider than a block": ([(3, 70)], 200, 1, 32, 64, 0, 0, 0),
    "eight key heads": ([(70, 70)], 8, 8, 64, 30, 0, 0, 0),
    "three key heads": ([(140, 140)], 6, 3, 96, 30, 1, 0, 0),
    "heads of 1": ([(70, 70)], 2, 1, 1, None, 0, 0, 0),
    "heads of 5": ([(70, 70)], 2, 1, 5, 30, 1, 0, 0),
    "heads of 65": ([(70, 140)], 2, 1, 65, None, 0, 0, 0),
    "heads of 80": ([(200, 200)], 4, 2, 80, 90, 4, 0, 0),
    "heads of 97": ([(40, 140)], 2, 2, 97, 60, 0, 0, 0),
    "heads of 120": ([(100, 140)], 2, 2, 120, 60, 0, 0, 0),
    "many sequences": ([(i % 5, i % 7 + 1) for i in range(200)], 2, 1, 32, 4, 1, 3, 3),
    "long": ([(1100, 1100)], 4, 1, 64, 300, 4, 0, 0),
}


def _case(name, dtype, **more):
    seqs, hq, hk, d, window, sinks, lead, tail = CASES[name]
    return Case(seqs, hq, hk, d, window, sinks, dtype, lead, tail, **more)


def _check_forward(c, y, lse, want, err):
    within("y", y, want["y"], err["y"], c.dtype)
    within("lse", lse, want["lse"], err["lse"], F)


def _check_backward(c, got, want, err, base=None):
    for a, v in zip("qkv", got):
        w, e = want[a + "b"], err[a + "b"]
        if base is not None:
            w = w + base[a].double()
        within(a + "b", v, w, e + 2 * U * w.abs(), c.dtype)


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("name", CASES)
def test_both_sweeps(name, dt):
    c = _case(name, dt)
    print(f"attention: {name} {IDS[dt]}", flush=True)
    want, err = formula(c)
    y, lse = c.forward()
    _check_forward(c, y, lse, want, err)
    got = c.backward(y, lse)
    _check_backward(c, got, want, err)
    # accumulated; and the same bits at every call
    g = gen(c.t)
    base = {a: normal(g, *getattr(c, a).shape, dtype=dt) for a in "qkv"}
    _check_backward(c, c.backward(y, lse, add=True, base=base), want, err, base)
    y2, lse2 = c.forward()
    assert torch.equal(y2, y) and torch.equal(lse2, lse)
    assert all(torch.equal(a, b) for a, b in zip(c.backward(y, lse), got))


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("name", ["window and sinks", "heads of 5", "heads of 80", "single tokens", "columns of none"])
def test_rows_apart(name, dt):
    """Rows apart at an odd offset, and parts of one wider matrix: the packed call's bits (straight and through registers)."""
    import stade_hip
    c = _case(name, dt)
    print(f"attention, rows apart: {name} {IDS[dt]}", flush=True)
    y, lse = c.forward()
    back = c.backward(y, lse)
    for gap in (3, 8):
        q, k, v, yb, yv = (apart(a.cuda(), gap) for a in (c.q, c.k, c.v, c.yb, torch.zeros_like(c.q)))
        lse2 = torch.empty_like(lse)
        stade_hip.attention(yv, lse2, q, k, v, *c.starts(), c.s, *c.size(), **c.form())
        assert torch.equal(yv, y) and torch.equal(lse2, lse)
        out = [apart(torch.zeros_like(a).cuda(), gap) for a in (c.q, c.k, c.v)]
        stade_hip.attention_b(yb, yv, lse2, q, out[0], k, out[1], v, out[2], *c.starts(), c.s, *c.size(), add=False, **c.form())
        assert all(torch.equal(a, b) for a, b in zip(out, back))
    # queries, keys and values side by side in one product's rows
    if c.t == c.tk:
        row = torch.cat([c.q, c.k, c.v], 1).cuda()
        a, b = c.hq * c.d, (c.hq + c.hk) * c.d
        y2, _ = c.forward(row[:, :a], row[:, a:b], row[:, b:])
        assert torch.equal(y2, y)


def test_parts_left_out():
    import stade_hip
    c = _case("window and sinks", B)
    y, lse = c.forward()
    y2 = torch.empty_like(y)
    stade_hip.attention(y2, None, c.q.cuda(), c.k.cuda(), c.v.cuda(), *c.starts(), c.s, *c.size(), **c.form())
    assert torch.equal(y2, y)
    whole = c.backward(y, lse)
    for parts in ("q", "k", "v", "qk", "kv", ""):
        for a, got, want in zip("qkv", c.backward(y, lse, parts=parts), whole):
            assert got is None if a not in parts else torch.equal(got, want)


@pytest.mark.parametrize("s", [0.0, -0.3, 2.0])
def test_factor_of_the_scores(s):
    c = _case("window and sinks", F, s=s)
    want, err = formula(c)
    y, lse = c.forward()
    _check_forward(c, y, lse, want, err)
    _check_backward(c, c.backward(y, lse), want, err)


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
def test_large_scores(dt):
    """Scores of some hundreds: the running maximum rises tile after tile, and most weights vanish."""
    c = _case("chunk of a long one", dt)
    c.k = (c.k.float() * torch.linspace(0.1, 8, c.tk)[:, None]).to(dt)
    c.q = (c.q.float() * 6).to(dt)
    want, err = formula(c)
    y, lse = c.forward()
    _check_forward(c, y, lse, want, err)
    _check_backward(c, c.backward(y, lse), want, err)


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
def test_values_that_are_not_finite_and_not_seen(dt):
    """Keys and values that no query sees (before the windows, and of no sequence) may hold anything."""
    c = Case([(1, 300), (40, 500), (3, 90)], 4, 2, 64, 30, 2, dt, lead=3, tail=70)
    want, err = formula(c)
    hidden = torch.ones(c.tk, dtype=torch.bool)
    for i, (nq, nk) in enumerate(c.seqs):
        hidden[c.ks[i]:c.ks[i] + nk] = ~c.seen(i).any(0)
    assert hidden.sum() > 400
    for a in (c.k, c.v):
        a[hidden] = float("nan")
        a[hidden.nonzero()[::2, 0]] = float("inf")
    c.q[:3] = c.yb[:3] = float("nan")    # columns of no sequence
    c.q[c.qs[-1]:] = c.yb[c.qs[-1]:] = float("inf")
    y, lse = c.forward()
    _check_forward(c, y, lse, want, err)
    kb, vb = c.backward(y, lse)[1:]
    for got, a in ((kb, "kb"), (vb, "vb")):
        assert not got.cpu()[hidden].any()
        within(a, got, want[a], err[a] + 2 * U * want[a].abs(), dt)
    qb = c.backward(y, lse, parts="q")[0]
    assert not qb[:3].any() and not qb[c.qs[-1]:].any()
    mine = slice(3, c.qs[-1])
    within("qb", qb[mine], want["qb"][mine], err["qb"][mine] + 2 * U * want["qb"][mine].abs(), dt)


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_finite_and_seen_by_some(dt, bad):
    """A value, key, query or shadow that is not finite reaches those that see it and no other, within a tile too."""
    c = Case([(200, 200), (70, 70)], 2, 1, 32, 45, 1, dt)
    want, err = formula(c)
    y0, lse0 = c.forward()
    at = 100
    sees = torch.zeros(c.t, dtype=torch.bool)
    sees[:200] = c.seen(0)[:, at]
    group = c.hq // c.hk

    def rows_of(m):
        return m.view(c.t, c.hq, c.d)

    # a value: column 3 of the rows that see it
    v = c.v.clone()
    c.v[at, 3] = bad
    y, lse = c.forward()
    off = ~torch.isfinite(rows_of(y)).cpu()
    assert torch.equal(off[..., 3], sees[:, None].expand(c.t, c.hq)) and not off[..., :3].any() and not off[..., 4:].any()
    clean = ~off.view(c.t, -1)
    within("y", y.cpu()[clean], want["y"][clean], err["y"][clean], dt)
    assert torch.isfinite(lse).all()
    qb, kb, vb = c.backward(y0, lse0)     # (what the forward sweep gave without it)
    assert torch.equal(~torch.isfinite(rows_of(qb)).all(-1).cpu(), sees[:, None].expand(c.t, c.hq))
    within("qb", qb.cpu()[~sees], want["qb"][~sees], (err["qb"] + 2 * U * want["qb"].abs())[~sees], dt)
    off = ~torch.isfinite(kb).cpu()
    assert off[at].all() and not off[:at].any() and not off[at + 1:].any()
    within("vb", vb, want["vb"], err["vb"] + 2 * U * want["vb"].abs(), dt)
    c.v = v

    # a query's shadow: its own row's qb, and the keys that it sees
    c.yb[at, 5] = bad
    qb, kb, vb = c.backward(y0, lse0)
    off = ~torch.isfinite(rows_of(qb)).cpu()
    assert off[at, 0].all() and off.sum() == c.d
    seen = torch.zeros(c.tk, dtype=torch.bool)
    seen[:200] = c.seen(0)[at]
    for got, a in ((kb, "kb"), (vb, "vb")):
        assert torch.equal(~torch.isfinite(got).all(-1).cpu(), seen)
        within(a, got.cpu()[~seen], want[a][~seen], (err[a] + 2 * U * want[a].abs())[~seen], dt)
    assert group == 2


def test_offsets_out_of_order():
    """Offsets that decrease or lie outside the columns raise the flag and are read as something within them."""
    import stade_hip
    c = _case("window and sinks", F)
    y, lse = torch.zeros(c.t, c.hq * c.d, device="cuda"), torch.zeros(c.t, c.hq, device="cuda")
    a = [v.cuda() for v in (c.q, c.k, c.v)]
    good = [torch.tensor(c.qs), torch.tensor(c.ks)]
    for which in range(2):
        for at, value in ((0, -1), (1, c.tk + 100), (2, 3), (3, 2 ** 40)):
            starts = [v.clone() for v in good]
            starts[which][at] = value
            with pytest.raises(stade_hip.StadeHipBoundsError):
                stade_hip.attention(y, lse, *a, *(v.cuda() for v in starts), c.s, *c.size(), check=True, **c.form())
            out = [torch.zeros_like(v) for v in a]
            with pytest.raises(stade_hip.StadeHipBoundsError):
                stade_hip.attention_b(c.yb.cuda(), y, lse, a[0], out[0], a[1], out[1], a[2], out[2], *(v.cuda() for v in starts), c.s, *c.size(), check=True,
                                      **c.form())
    stade_hip.attention(y, lse, *a, *(v.cuda() for v in good), c.s, *c.size(), check=True, **c.form())


def test_nothing_to_do():
    import stade_hip
    e, l, one = torch.empty(0, 8, device="cuda"), torch.empty(0, 2, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    stade_hip.attention(e, l, e, e, e, one, one, 1.0, 4, 2, 2, 0, 0, 0)
    k = torch.ones(5, 8, device="cuda")
    kb = torch.ones(5, 8, device="cuda")
    stade_hip.attention(e, l, e, k, k, one, one, 1.0, 4, 2, 2, 0, 5, 0)
    stade_hip.attention_b(e, e, l, e, e, k, kb, k, None, one, one, 1.0, 4, 2, 2, 0, 5, 0)
    assert kb.eq(1).all()
    stade_hip.attention_b(e, e, l, e, e, k, kb, k, None, one, one, 1.0, 4, 2, 2, 0, 5, 0, add=False)
    assert not kb.any()
    # queries and no keys at all
    q, y, lse, qb = torch.ones(3, 8, device="cuda"), torch.ones(3, 8, device="cuda"), torch.ones(3, 2, device="cuda"), torch.ones(3, 8, device="cuda")
    at, none = torch.tensor([0, 3]).cuda(), torch.zeros(2, dtype=torch.int64, device="cuda")
    stade_hip.attention(y, lse, q, e, e, at, none, 1.0, 4, 2, 2, 3, 0, 1)
    assert not y.any() and torch.isneginf(lse).all()
    stade_hip.attention_b(q, y, lse, q, qb, e, e, e, e, at, none, 1.0, 4, 2, 2, 3, 0, 1, add=False)
    assert not qb.any()


@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_gradient_by_differences(which):
    """The directional derivative of <yb, attention> by differences of the forward kernel."""
    c = Case([(40, 40), (9, 70)], 2, 1, 16, 20, 2, F)
    want, err = formula(c)
    y, lse = c.forward()
    got = dict(zip("qkv", c.backward(y, lse)))[which].double().cpu()
    dx, h = normal(gen(5), *getattr(c, which).shape), 2.0 ** -6
    at, slack, plain = [], 0.0, []
    here = getattr(c, which)
    for e in (h, -h):
        setattr(c, which, here + e * dx)
        w, er = formula(c, grads=False)
        at.append((c.yb.double() * c.forward()[0].double().cpu()).sum())
        plain.append((c.yb.double() * w["y"]).sum())
        slack += (c.yb.double().abs() * (er["y"] + U * w["y"].abs())).sum()
    setattr(c, which, here)
    exact = (want[which + "b"] * dx.double()).sum()
    bound = ((err[which + "b"] + U * want[which + "b"].abs()) * dx.double().abs()).sum()
    assert abs((got * dx.double()).sum() - exact) <= bound
    # the differences' own curvature, and the forward kernel's errors over the step
    assert abs((at[0] - at[1]) / (2 * h) - exact) <= abs((plain[0] - plain[1]) / (2 * h) - exact) + slack / (2 * h)
