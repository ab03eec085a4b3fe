"""The adjoint of attention in f16 at the ends: gradients that are 0 but for rounding, and shadows so small that only large keys
or queries make values of them."""
import pytest
import torch
from attnhelp import Case
from lmhelp import U, within

pytestmark = pytest.mark.gpu
H = torch.float16


@pytest.mark.parametrize("seqs,window", [([(300, 300), (70, 90)], 1), ([(1, 1)] * 50, None)], ids=["a window of one", "one key each"])
@pytest.mark.parametrize("d", [64, 128])
def test_one_key_a_query(seqs, window, d):
    """P is 1 and S 0: what is left of yb v^T - delta are roundings.  Of P: the score's, lse's (10 U and its size's), the exponent's
    with 14 added, twice (5 U each), and the exponential's; and of a product's d terms."""
    c = Case(seqs, 4, 2, d, window, 0, H)
    y, lse = c.forward()
    qb, kb, vb = c.backward(y, lse)
    own = torch.cat([torch.arange(c.ks[i] + nk - nq, c.ks[i] + nk) for i, (nq, nk) in enumerate(seqs)])
    heads = lambda m, n: m.double().view(-1, n, d)   # noqa: E731
    q, yb = heads(c.q, 4), heads(c.yb, 4)
    k, v = (heads(m, 2)[own].repeat_interleave(2, 1) for m in (c.k, c.v))
    score = c.s * (q.abs() * k.abs()).sum(-1, keepdim=True)
    g = (yb.abs() * v.abs()).sum(-1, keepdim=True)
    s = ((d + 10) * U * score + 30 * U) * g + 2 * (d + 4) * U * g
    within("qb", qb, torch.zeros(c.t, 4 * d), (c.s * s * k.abs()).flatten(1), H)
    want = torch.zeros(c.tk, 2, d, dtype=torch.float64)
    want.index_add_(0, own, (c.s * s * q.abs()).view(c.t, 2, 2, d).sum(2))
    within("kb", kb, torch.zeros(c.tk, 2 * d), want.flatten(1), H)


def test_shadows_that_large_keys_make_values_of():
    """Two keys, of which a query sees both alike: S = P (g - delta) with P = 1 / 2 is +- (g0 - g1) / 4, here 2^-46 and 2^-50; times
    a thousand queries (or a key) of 2^15 that is a value of f16."""
    for power in (-46, -50):
        n = 8192
        c = Case([(n, n + 1)], 1, 1, 8, 0, 2, H, s=1.0)      # (sinks alone: two keys are seen by all)
        c.q.zero_(), c.k.zero_(), c.v.zero_(), c.yb.zero_()
        c.q[:, 0] = 32768.0
        c.k[0, 1] = c.k[1, 1] = 32768.0                          # (scores of 0, and lse = log 2)
        c.yb[:, 2] = 2.0 ** -24
        c.v[0, 2] = 2.0 ** (power + 24 + 2)
        y, lse = c.forward()
        # y = v / 2 is not a value of f16 where it is below 2^-24: delta for kb is the sum of P yb v^T
        qb, kb, vb = (a.cpu().double() for a in c.backward(y, lse))
        want = n * 2.0 ** power * 32768.0
        assert abs(kb[0, 0] - want) <= (2.0 ** -10 + n * U) * want + 2.0 ** -25, (float(kb[0, 0]), want)
        assert abs(kb[1, 0] + want) <= (2.0 ** -10 + n * U) * want + 2.0 ** -25, (float(kb[1, 0]), want)
        # the two keys' parts of qb go against each other
        assert not qb.any() and not kb[:, 1:].any()
        assert abs(vb[0, 2] - n * 2.0 ** -25) <= (2.0 ** -10 + n * U) * n * 2.0 ** -25
