"""Attention in f16, weights far below the largest: one weight of 1 among many thousands of 2^-25.5, which make up the result."""
import attnhelp
import pytest
import torch
from attnhelp import Case, formula
from lmhelp import within

pytestmark = pytest.mark.gpu
H = torch.float16


@pytest.mark.parametrize("heads", [1, 64])      # (64: as many rows' tiles as take their keys in one block each)
@pytest.mark.parametrize("where", ["first", "last"])
def test_many_small_weights(heads, where, monkeypatch):
    n = 30000
    c = Case([(1, n)] + [(1, 1)] * 15, heads, heads, 8, None, 0, H, s=1.0)
    at = 0 if where == "first" else n - 1
    c.q.zero_()
    c.k.zero_()
    c.q[:, ::8] = 1
    c.k[at, ::8] = 17.6875          # weights of the others: exp(-17.6875) = 2^-25.5
    c.v = (c.v.float().abs() + 0.5).to(H)
    c.v[at] = 0
    # Weights are held in steps of 2^-31 of the largest: 2^-24 where 1 stands for 2^7
    monkeypatch.setattr(attnhelp, "LEAST", {**attnhelp.LEAST, H: 2.0 ** -31})
    want, err = formula(c, grads=False)
    assert (err["y"][0] < 0.1 * want["y"][0].abs()).all() and (want["y"][0] > 2.0 ** -12).all()
    y, lse = c.forward()
    within("y", y, want["y"], err["y"], H)
    within("lse", lse, want["lse"], err["lse"], torch.float32)
