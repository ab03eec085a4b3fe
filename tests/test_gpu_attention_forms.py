"""Attention in the forms that longer calls take: keys over several blocks, and tiles of keys whose rows go over several blocks."""
import pytest
import torch

from attnhelp import Case, formula
from lmhelp import IDS, TYPES, U, gen, normal, within

pytestmark = pytest.mark.gpu
BF = torch.bfloat16

# few rows and many keys: over several blocks each
SPLIT = {
    "one token": ([(1, 9000)], 8, 2, 64, None, 0),
    "tokens of different lengths": ([(1, 5000), (1, 3), (1, 0), (0, 70), (1, 2500), (2, 1025)], 4, 1, 80, None, 0),
    "chunks": ([(70, 3000), (130, 1500)], 6, 2, 128, None, 0),
    "a window over blocks": ([(3, 6000), (1, 4000)], 2, 2, 32, 2500, 5),
    "heads that divide nothing": ([(1, 4000), (5, 2100)], 3, 3, 40, None, 0),
}


def _forward(c, want, err):
    y, lse = c.forward()
    within("y", y, want["y"], err["y"], c.dtype)
    within("lse", lse, want["lse"], err["lse"], torch.float32)
    return y, lse


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("name", SPLIT)
def test_keys_over_blocks(name, dt):
    seqs, hq, hk, d, window, sinks = SPLIT[name]
    c = Case(seqs, hq, hk, d, window, sinks, dt, lead=2, tail=3)
    want, err = formula(c, grads=False)
    print(f"keys over blocks: {name} {IDS[dt]}", flush=True)
    y, lse = _forward(c, want, err)
    y2, lse2 = c.forward()
    assert torch.equal(y, y2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
def test_keys_over_blocks_not_finite(dt, bad):
    """Keys and values that no query sees may hold anything; a value that one sees reaches its column alone."""
    c = Case([(1, 4000), (2, 3000)], 4, 2, 64, 1500, 3, dt, tail=100)
    want, err = formula(c, grads=False)
    hidden = torch.ones(c.tk, dtype=torch.bool)
    for i in range(2):
        hidden[c.ks[i]:c.ks[i + 1]] = ~c.seen(i).any(0)
    assert hidden.sum() > 3000
    c.k[hidden], c.v[hidden] = bad, bad
    print(f"keys over blocks, not finite: {IDS[dt]} {bad}", flush=True)
    _forward(c, want, err)
    c.v[3500, 70] = bad      # sequence 0, key head 1, column 6
    y, lse = c.forward()
    off = ~torch.isfinite(y).cpu().view(c.t, c.hq, c.d)
    assert off[0, 2:, 6].all() and off.sum() == 2
    within("y", y.cpu()[~off.view(c.t, -1)], want["y"][~off.view(c.t, -1)], err["y"][~off.view(c.t, -1)], dt)
    c.k[3500, :] = bad       # (scores of NaN, or of infinities of either sign)
    y, lse = c.forward()
    assert not torch.isfinite(lse[0]).any() or not torch.isfinite(y[0]).all()
    within("y", y[1:], want["y"][1:], err["y"][1:], dt)
    within("lse", lse[1:], want["lse"][1:], err["lse"][1:], torch.float32)


# few keys and many rows: the rows that see a tile go over several blocks, whose sums are joined
JOINED = {
    "one tile": ([(500, 100)], 8, 1, 64, None, 0),
    "short ones": ([(300, 300), (1, 200), (700, 700)], 6, 2, 80, None, 0),
    "with sinks": ([(900, 900), (40, 50)], 4, 2, 128, 300, 7),
    "many sinks": ([(1200, 1200)], 2, 1, 24, 64, 64),
    # many rows past the window that see the sinks: in blocks of their own
    "far rows": ([(1500, 1500)], 4, 1, 64, 100, 4),
    "far rows of several": ([(2000, 2100), (700, 700), (1, 5), (0, 9)], 4, 2, 128, 64, 9),
    "far rows, sinks past 32": ([(1300, 1300)], 2, 2, 40, 30, 40),
    "far rows of one among short ones": ([(5, 5)] * 40 + [(1100, 1100)], 8, 1, 80, 20, 3),
    "few far rows of one among short ones": ([(5, 5)] * 40 + [(700, 700)], 8, 1, 80, 20, 3),
}


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("name", JOINED)
def test_rows_over_blocks(name, dt):
    seqs, hq, hk, d, window, sinks = JOINED[name]
    c = Case(seqs, hq, hk, d, window, sinks, dt, lead=1, tail=2)
    want, err = formula(c)
    print(f"rows over blocks: {name} {IDS[dt]}", flush=True)
    y, lse = _forward(c, want, err)
    g = gen(c.t)
    base = {a: normal(g, *getattr(c, a).shape, dtype=dt) for a in "qkv"}
    first = None
    for add in (False, True, False):
        got = c.backward(y, lse, add=add, base=base)
        for a, v in zip("qkv", got):
            w, e = want[a + "b"], err[a + "b"]
            within(a + "b", v, w + base[a].double() if add else w, e + 2 * U * w.abs(), dt)
        if not add:
            assert first is None or all(torch.equal(u, v) for u, v in zip(first, got))
            first = got


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
def test_past_the_rounds_of_the_card(dt):
    """More tiles of keys than the card has places: whole rounds, and the rest of them split."""
    c = Case([(40, 40)] * 70 + [(1, 1), (600, 600)], 8, 4, 32, None, 0, dt)
    want, err = formula(c)
    print(f"many sequences {IDS[dt]}", flush=True)
    y, lse = _forward(c, want, err)
    for a, v in zip("qkv", c.backward(y, lse)):
        within(a + "b", v, want[a + "b"], err[a + "b"] + 2 * U * want[a + "b"].abs(), dt)


@pytest.mark.parametrize("s", [0.0, 1e-42, -1e-30, -0.7])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("seqs", [[(400, 400), (5, 5), (260, 300)], [(1, 4096), (1, 64)], [(64, 64), (1, 128)]], ids=str)
def test_factors_that_leave_no_scores(seqs, dt, s):
    """Scores of 0 or nearly: equal weights, also over whole tiles of keys and over several blocks."""
    c = Case(seqs, 4, 1, 128, 70 if seqs[0][0] == 400 else None, 4, dt, s=s)
    want, err = formula(c)
    print(f"factor {s} {IDS[dt]}", flush=True)
    y, lse = _forward(c, want, err)
    # s is taken in fp32: qb and kb, multiples of it, are off by its rounding, for 1e-42 by up to 2^-150 / 1e-42 = 7e-4 of them
    off = abs(float(torch.tensor(s, dtype=torch.float32)) - s) / abs(s) if s else 0.0
    for a, v in zip("qkv", c.backward(y, lse)):
        within(a + "b", v, want[a + "b"], err[a + "b"] + (2 * U + off) * want[a + "b"].abs(), dt)
