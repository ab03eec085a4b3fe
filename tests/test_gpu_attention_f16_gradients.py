"""The adjoint of attention in f16 where its factors are far from 1: shadows that are small or large, and weights of long sequences.
P and S = P (yb v^T - delta) are products' factors in f16, held to half steps of 2^-36 of the largest S of a row (for qb) or of a block's rows."""
import attnhelp
import pytest
import torch
from attnhelp import Case, formula
from lmhelp import U, gen, within

pytestmark = pytest.mark.gpu
H = torch.float16
SHAPES = {"a long one": ([(2100, 2100)], 2, 1, 64, None, 0), "window and sinks": ([(1500, 1500), (40, 300)], 2, 1, 128, 700, 4),
          "heads of 40": ([(30, 3000), (1200, 1200)], 4, 2, 40, None, 0), "rows through registers": ([(900, 1700)], 2, 2, 35, None, 0),
          "far rows": ([(2500, 2500)], 2, 1, 64, 300, 40)}


def _bounds(c, least, monkeypatch):
    """The formula's bounds with factors held in steps of `least`."""
    with monkeypatch.context() as m:
        m.setattr(attnhelp, "LEAST", {**attnhelp.LEAST, H: least})
        return formula(c)[1]


def _case(name, scale_q, scale_k):
    seqs, hq, hk, d, window, sinks = SHAPES[name]
    c = Case(seqs, hq, hk, d, window, sinks, H, lead=1, tail=2)
    c.q, c.k = (c.q.float() * scale_q).to(H), (c.k.float() * scale_k).to(H)
    return c


@pytest.mark.parametrize("part", ["q", "k"])
@pytest.mark.parametrize("name", SHAPES)
def test_small_shadows(name, part, monkeypatch):
    """Shadows of 2^-22, over some thousand keys: S is 2^-30 and less."""
    c = _case(name, *((2.0 ** -10, 2.0 ** 10) if part == "q" else (2.0 ** 10, 2.0 ** -10)))
    c.yb = (c.yb.float() * 2.0 ** -22).to(H)
    want, _ = formula(c)
    # S is held to 2^-36 of the largest, which here is below 2^-17
    w = want[part + "b"]
    err = _bounds(c, 2.0 ** -53, monkeypatch)[part + "b"] + 2 * U * w.abs()
    assert (err + 2.0 ** -24 < 0.8 * w.abs()).float().mean() > 0.3      # (the bound tells a result from none, and the type holds it)
    got = c.backward(*c.forward())["qk".index(part)]
    within(part + "b", got, w, err, H)


@pytest.mark.parametrize("name", SHAPES)
def test_large_shadows(name, monkeypatch):
    """S past 65504, of finite operands with finite results."""
    c = _case(name, 2.0 ** -6, 2.0 ** -8)
    c.yb, c.v = (c.yb.float() * 2.0 ** 10).to(H), (c.v.float() * 2.0 ** 8).to(H)
    want, _ = formula(c)
    y, lse = c.forward()
    got = c.backward(y, lse)
    for a, v, least in zip("qkv", got, (2.0 ** -14, 2.0 ** -14, 2.0 ** -38)):    # (S is below 2^22, and held to 2^-36 of that; P to 2^-39)
        within(a + "b", v, want[a + "b"], _bounds(c, least, monkeypatch)[a + "b"] + 2 * U * want[a + "b"].abs(), H)
    assert all(torch.equal(u, v) for u, v in zip(got, c.backward(y, lse)))


@pytest.mark.parametrize("name", SHAPES)
def test_rows_of_many_sizes(name):
    """Shadows from 2^-22 to 2^12 in one sequence, small rows first and last: each row's qb and each key's sums to their own bounds."""
    c = _case(name, 1.0, 1.0)
    power = torch.randint(-22, 13, (c.t, 1), generator=gen(3)).float()
    c.yb = (c.yb.float() * torch.exp2(power)).to(H)
    want, err = formula(c)
    y, lse = c.forward()
    for a, got in zip("qkv", c.backward(y, lse)):
        within(a + "b", got, want[a + "b"], err[a + "b"] + 2 * U * want[a + "b"].abs(), H)


def test_small_weights_of_values(monkeypatch):
    """Every other key has weights of exp(-12) of the others', 2^-26 and less: their vb alone."""
    c = Case([(2400, 2400)], 1, 1, 64, None, 0, H)
    c.q[:, 0], c.k[:, 0], c.k[1::2, 0] = 4, 0, -24
    c.yb = (1 + c.yb.float().abs()).mul(2.0 ** 9).to(H)
    want, _ = formula(c)
    err = _bounds(c, 2.0 ** -38, monkeypatch)     # (P is held to 2^-39)
    small = torch.arange(1501, 2300, 2)
    assert (want["vb"][small] > 2.0 ** -12).all() and (err["vb"][small] < 0.2 * want["vb"][small]).all()
    vb = c.backward(*c.forward())[2]
    within("vb", vb, want["vb"], err["vb"] + 2 * U * want["vb"].abs(), H)
