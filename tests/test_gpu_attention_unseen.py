"""Rows that see nothing beside keys, values and queries that are not finite: zeros and -Inf, whatever a tile holds.  And keys that are not
finite where the keys of a row go over several blocks."""
import pytest
import torch

from attnhelp import Case, formula
from lmhelp import IDS, TYPES, U, within

pytestmark = pytest.mark.gpu
BAD = [float("nan"), float("inf"), -float("inf")]
# more queries than keys, so that the first queries see nothing; straight loads and through registers, and several blocks of rows
SHAPES = {"heads of 64": (4, 2, 64), "heads of 5": (2, 1, 5), "heads of 128": (6, 1, 128)}


def _case(name, dt):
    hq, hk, d = SHAPES[name]
    return Case([(40, 20), (150, 60), (7, 7)], hq, hk, d, dtype=dt)


def _rows_that_see(c, key):
    """Truth values of the columns of c whose queries see column `key` of the keys, and of those that see anything."""
    sees, some = torch.zeros(c.t, dtype=torch.bool), torch.zeros(c.t, dtype=torch.bool)
    for i, (nq, nk) in enumerate(c.seqs):
        ok = c.seen(i)
        some[c.qs[i]:c.qs[i] + nq] = ok.any(1)
        if c.ks[i] <= key < c.ks[i] + nk:
            sees[c.qs[i]:c.qs[i] + nq] = ok[:, key - c.ks[i]]
    return sees, some


def _nothing(c, y, lse, some):
    assert not y.cpu()[~some].any() and torch.isneginf(lse.cpu()[~some]).all()


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("name", SHAPES)
def test_rows_that_see_nothing(name, dt, bad):
    c = _case(name, dt)
    want, err = formula(c)
    y0, lse0 = c.forward()
    print(f"rows that see nothing: {name} {IDS[dt]} {bad}", flush=True)
    for key in (10, 20 + 33):           # of the first and the second sequence
        sees, some = _rows_that_see(c, key)
        assert (~some).sum() == 20 + 90 and sees.any()
        clean = ~sees
        # a value: one column of those that see it
        v = c.v.clone()
        c.v[key, 3] = bad
        y, lse = c.forward()
        _nothing(c, y, lse, some)
        within("y", y.cpu()[clean], want["y"][clean], err["y"][clean], dt)
        within("lse", lse, want["lse"], err["lse"], torch.float32)
        assert not torch.isfinite(y.cpu()[sees].view(-1, c.hq, c.d)[:, 0, 3]).any()
        qb, kb, vb = c.backward(y0, lse0)
        assert not qb.cpu()[~some].any()
        within("qb", qb.cpu()[clean], want["qb"][clean], (err["qb"] + 2 * U * want["qb"].abs())[clean], dt)
        other = torch.arange(c.tk) != key
        within("kb", kb.cpu()[other], want["kb"][other], (err["kb"] + 2 * U * want["kb"].abs())[other], dt)
        within("vb", vb, want["vb"], err["vb"] + 2 * U * want["vb"].abs(), dt)
        c.v = v
        # a key
        k = c.k.clone()
        c.k[key] = bad
        y, lse = c.forward()
        _nothing(c, y, lse, some)
        within("y", y.cpu()[clean], want["y"][clean], err["y"][clean], dt)
        within("lse", lse.cpu()[clean], want["lse"][clean], err["lse"][clean], torch.float32)
        c.k = k
    # a query that sees nothing and one that sees: its own row, and a query of nothing stays one
    q = c.q.clone()
    some = _rows_that_see(c, 0)[1]
    c.q[5] = c.q[30] = bad
    y, lse = c.forward()
    _nothing(c, y, lse, some)
    own = torch.arange(c.t) != 30
    within("y", y.cpu()[own], want["y"][own], err["y"][own], dt)
    c.q = q


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
def test_nothing_seen_at_all(dt, bad):
    """A window of none without sinks: zeros and -Inf and no gradients, of operands that hold nothing finite."""
    c = Case([(60, 60), (1, 300)], 2, 1, 16, 0, 0, dt)
    for a in (c.q, c.k, c.v):
        a.fill_(bad)
    y, lse = c.forward()
    assert not y.any() and torch.isneginf(lse).all()
    assert not any(g.any() for g in c.backward(y, lse))


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
def test_scores_of_minus_infinity_alone(dt):
    """Rows all of whose scores are -Inf: zeros and -Inf, of few keys as of many."""
    for nk in (3, 5000):
        c = Case([(1, nk), (1, 4)], 2, 1, 16, None, 0, dt)
        c.q[0], c.k[:nk] = 1, 0
        c.k[:nk, 2] = -float("inf")
        want, err = formula(Case([(1, nk), (1, 4)], 2, 1, 16, None, 0, dt), grads=False)
        y, lse = c.forward()
        assert not y[0].any() and torch.isneginf(lse[0]).all()
        within("y", y[1:], want["y"][1:], err["y"][1:], dt)
        within("lse", lse[1:], want["lse"][1:], err["lse"][1:], torch.float32)


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
def test_keys_that_are_seen_over_blocks(dt, bad):
    """A key of a token whose keys go over several blocks: scores of NaN reach all of a head's row; scores of -Inf take the key out."""
    c = Case([(1, 4000), (2, 3000)], 4, 2, 64, 1500, 3, dt, tail=100)
    want, err = formula(c, grads=False)
    at, k = 3500, c.k.clone()
    c.k[at] = float("nan")
    y, lse = c.forward()
    assert torch.isnan(y[0]).all() and torch.isnan(lse[0]).all()
    within("y", y[1:], want["y"][1:], err["y"][1:], dt)
    # one value of the key alone: the score is `bad` by the sign of the query's value (as it multiplies it)
    c.k = k.clone()
    c.k[at, ::c.d] = bad
    print(f"a key over blocks: {IDS[dt]} {bad}", flush=True)
    y, lse = (a.cpu() for a in c.forward())
    within("y", y[1:], want["y"][1:], err["y"][1:], dt)
    within("lse", lse[1:], want["lse"][1:], err["lse"][1:], torch.float32)
    seen = 0
    for h in range(c.hq):
        cols, kv = slice(h * c.d, (h + 1) * c.d), slice(h // 2 * c.d, (h // 2 + 1) * c.d)
        score = c.q[0, h * c.d].double() * bad
        if score != -float("inf"):
            assert not torch.isfinite(y[0, cols]).any() and not torch.isfinite(lse[0, h])
            continue
        # (y - p v) / (1 - p) without the key: its bound is at most twice the whole row's, by the parts of which it is made
        p = torch.exp(c.s * (c.q[0, cols].double() @ k[at, kv].double()) - want["lse"][0, h])
        assert p < 0.02
        within("y", y[0, cols], (want["y"][0, cols] - p * c.v[at, kv].double()) / (1 - p), 2.1 * err["y"][0, cols], dt)
        within("lse", lse[0, h:h + 1], (want["lse"][0, h] + torch.log1p(-p))[None], 2.1 * err["lse"][0, h:h + 1], torch.float32)
        seen += 1
    assert seen or bad != bad or not torch.isfinite(y[0]).any()
