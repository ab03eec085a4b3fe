"""expert_order, expert_take, expert_join and their adjoints against loops over the slots in 64 bits."""
import pytest
import torch

from lmhelp import IDS, TYPES, U, apart, gen, normal, within

pytestmark = pytest.mark.gpu

# (tokens, slots, experts, columns)
SIZES = [(1, 1, 1, 1), (5, 2, 3, 7), (3, 8, 4, 8), (40, 3, 60, 9), (77, 4, 30, 1111), (300, 2, 8, 512), (130, 5, 16, 513), (9, 64, 300, 40), (3000, 2, 64, 96), (2, 1, 2, 5000)]


def _ids(t, k, e, g, dropped=0.1):
    ids = torch.randint(1, e + 1, (t, k), generator=g)
    return torch.where(torch.rand(t, k, generator=g) < dropped, torch.zeros_like(ids), ids)


def _order(ids, e):
    """(order, place, start) by a stable sort in plain Python."""
    flat = ids.flatten().tolist()
    order = sorted(range(len(flat)), key=lambda i: (flat[i] == 0, flat[i], i))
    place = [0] * len(flat)
    for j, i in enumerate(order):
        place[i] = j + 1 if flat[i] else 0
    start = [sum(1 for v in flat if 0 < v <= b) for b in range(e + 1)]
    return torch.tensor([i + 1 for i in order]), torch.tensor(place).reshape(ids.shape), torch.tensor(start)


def _arrays(t, k, e):
    new = lambda *n: torch.full(n, -7, dtype=torch.int64, device="cuda")   # noqa: E731
    return new(t * k), new(t, k), new(e + 1)


@pytest.mark.parametrize("size", SIZES + [(20000, 2, 100, 1), (50, 2, 4096, 1)], ids=str)
def test_order(size):
    import stade_hip
    t, k, e, _ = size
    ids = _ids(t, k, e, gen(t))
    order, place, start = _arrays(t, k, e)
    print(f"expert_order {size}", flush=True)
    stade_hip.expert_order(ids.cuda(), order, place, start, k, e, t, check=True)
    for got, want in zip((order, place, start), _order(ids, e)):
        assert torch.equal(got.cpu(), want)


def _gather(rows, place):
    """(t, k, d): the rows at the places, zeros for none."""
    return torch.where((place > 0)[..., None], rows[(place - 1).clamp_min(0)], torch.zeros((), dtype=rows.dtype))


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_rows(size, dt):
    import stade_hip
    t, k, e, d = size
    g = gen(t + d)
    _, place, start = _order(_ids(t, k, e, g), e)
    p = torch.rand(t, k, generator=g)
    x, ys, xsb, yb = normal(g, t, d, dtype=dt), *(normal(g, t * k, d, dtype=dt) for _ in range(2)), normal(g, t, d, dtype=dt)
    at, P = place.cuda(), p.cuda()
    here = int(start[-1])
    print(f"expert rows {size} {IDS[dt]}", flush=True)

    # take: exact, and the columns behind the last expert's as they were
    xs = torch.full((t * k, d), 5.0, dtype=dt, device="cuda")
    stade_hip.expert_take(xs, x.cuda(), at, d, k, t, check=True)
    want = torch.full((t * k, d), 5.0, dtype=dt)
    token = torch.arange(t)[:, None].expand(t, k)
    want[place[place > 0] - 1] = x[token[place > 0]]
    assert torch.equal(xs.cpu(), want) and (xs[here:] == 5.0).all()
    xv = apart(torch.full((t * k, d), 5.0, dtype=dt, device="cuda"))
    stade_hip.expert_take(xv, apart(x.cuda()), at, d, k, t)
    assert torch.equal(xv, xs)

    ysd, xsd, ybd = ys.double(), xsb.double(), yb.double()
    for add in (False, True):
        base = normal(gen(d), t, d, dtype=dt)
        b = base.double() if add else torch.zeros(t, d, dtype=torch.float64)

        def start_of(v):
            return v.cuda() if add else torch.full_like(v, float("nan")).cuda()

        # k terms and what was there, one after the other
        for name, rows, w in (("join", ysd, p), ("join without weights", ysd, None), ("take_b", xsd, None)):
            terms = _gather(rows, place) * (1.0 if w is None else w.double()[..., None])
            y = start_of(base)
            if name == "take_b":
                stade_hip.expert_take_b(xsb.cuda(), y, at, d, k, t, add=add, check=True)
            else:
                stade_hip.expert_join(y, ys.cuda(), None if w is None else P, at, d, k, t, add=add, check=True)
            within(name, y, b + terms.sum(1), (k + 1) * U * (b.abs() + terms.abs().sum(1)), dt)
            yv = apart(start_of(base))
            if name == "take_b":
                stade_hip.expert_take_b(apart(xsb.cuda()), yv, at, d, k, t, add=add)
            else:
                stade_hip.expert_join(yv, apart(ys.cuda()), None if w is None else P, at, d, k, t, add=add)
            assert torch.equal(yv, y)

        rows0, pb0 = normal(gen(d + 1), t * k, d, dtype=dt), normal(gen(3), t, k)
        ysb, pb = rows0.cuda(), start_of(pb0)
        stade_hip.expert_join_b(yb.cuda(), ys.cuda(), ysb, P, pb, at, d, k, t, add=add, check=True)
        want = rows0.double()
        v = (p.double()[..., None] * ybd[:, None])[place > 0]
        old = want[place[place > 0] - 1].clone() if add else torch.zeros_like(v)
        want[place[place > 0] - 1] = old + v
        slack = torch.zeros_like(want)
        slack[place[place > 0] - 1] = 2 * U * (old.abs() + v.abs())
        within("ysb", ysb[:here], want[:here], slack[:here], dt)
        assert torch.equal(ysb[here:].cpu(), rows0[here:])
        terms = _gather(ysd, place) * ybd[:, None]
        b = pb0.double() if add else torch.zeros(t, k, dtype=torch.float64)
        # 8 values a lane in each 512 columns, six steps over the wave, and what was there
        within("pb", pb, b + terms.sum(-1), (8 * (d // 512 + 1) + 8) * U * (terms.abs().sum(-1) + b.abs()), torch.float32)
        only, alone = start_of(pb0), rows0.cuda()
        stade_hip.expert_join_b(yb.cuda(), ys.cuda(), None, P, only, at, d, k, t, add=add)
        stade_hip.expert_join_b(yb.cuda(), None, alone, P, None, at, d, k, t, add=add)
        assert torch.equal(only, pb) and torch.equal(alone, ysb)
        # its rows' shadow in the rows' place
        same, pb2 = ys.cuda(), start_of(pb0)
        if not add:
            stade_hip.expert_join_b(yb.cuda(), same, same, P, pb2, at, d, k, t, add=False)
            assert torch.equal(pb2, pb) and torch.equal(same[:here], ysb[:here])


def test_ids_and_places_out_of_range():
    """An id of no expert, and a place of no row, are taken as none and raise the flag."""
    import stade_hip
    t, k, e, d = 6, 2, 3, 16
    ids = torch.tensor([[1, 4], [2, -1], [3, 1], [0, 2], [1, 1], [9, 3]])
    order, place, start = _arrays(t, k, e)
    with pytest.raises(stade_hip.StadeHipBoundsError):
        stade_hip.expert_order(ids.cuda(), order, place, start, k, e, t, check=True)
    want = _order(torch.where((ids > 0) & (ids <= e), ids, torch.zeros_like(ids)), e)
    assert torch.equal(place.cpu(), want[1]) and torch.equal(start.cpu(), want[2])
    bad = want[1].clone()
    bad[0, 0], bad[3, 1] = 13, -5
    good = torch.where((bad < 0) | (bad > t * k), torch.zeros_like(bad), bad)
    x, ys, p = normal(gen(1), t, d).cuda(), normal(gen(2), t * k, d).cuda(), torch.rand(t, k).cuda()

    def calls(at, check):
        xs, y, xb, ysb, pb = torch.zeros(t * k, d).cuda(), x.clone(), x.clone(), torch.zeros(t * k, d).cuda(), p.clone()
        out = []
        for f in (lambda: stade_hip.expert_take(xs, x, at, d, k, t, check=check), lambda: stade_hip.expert_join(y, ys, p, at, d, k, t, check=check),
                  lambda: stade_hip.expert_take_b(ys, xb, at, d, k, t, check=check),
                  lambda: stade_hip.expert_join_b(x, ys, ysb, p, pb, at, d, k, t, check=check)):
            if check:
                with pytest.raises(stade_hip.StadeHipBoundsError):
                    f()
            else:
                f()
        return [xs, y, xb, ysb, pb]

    assert all(torch.equal(a, b) for a, b in zip(calls(bad.cuda(), True), calls(good.cuda(), False)))


def test_nothing_to_do():
    import stade_hip
    e, i = torch.empty(0, 4, device="cuda"), torch.empty(0, 2, dtype=torch.int64, device="cuda")
    start = torch.full((4,), -7, dtype=torch.int64, device="cuda")
    stade_hip.expert_order(i, i.flatten(), i, start, 2, 3, 0)
    assert not start.any()
    stade_hip.expert_take(e, e, i, 4, 2, 0)
    stade_hip.expert_join(e, e, None, i, 4, 2, 0)
    stade_hip.expert_take_b(e, e, i, 4, 2, 0)
    stade_hip.expert_join_b(e, e, e, None, None, i, 4, 2, 0)
    # no slots: set to zeros, accumulated as it is
    y, none = torch.ones(3, 4, device="cuda"), torch.empty(3, 0, dtype=torch.int64, device="cuda")
    stade_hip.expert_join(y, e, None, none, 4, 0, 3, add=True)
    assert y.eq(1).all()
    stade_hip.expert_join(y, e, None, none, 4, 0, 3)
    assert not y.any()
    # all slots without an expert
    ids = torch.zeros(3, 2, dtype=torch.int64, device="cuda")
    order, place, start = _arrays(3, 2, 3)
    stade_hip.expert_order(ids, order, place, start, 2, 3, 3)
    assert not place.any() and not start.any()
    y, ys, pb = torch.ones(3, 4, device="cuda"), torch.full((6, 4), float("nan"), device="cuda"), torch.ones(3, 2, device="cuda")
    stade_hip.expert_join(y, ys, None, place, 4, 2, 3)
    stade_hip.expert_join_b(y, ys, None, None, pb, place, 4, 2, 3, add=False)
    assert not y.any() and not pb.any()
