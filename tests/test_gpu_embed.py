"""embed, embed_b and token_order against plain references in 64 bits."""
import pytest
import torch

from lmhelp import IDS, ROUND, TYPES, U, apart, cuda, gen, normal, within

pytestmark = pytest.mark.gpu


def _tokens(g, t, v, kind):
    if v == 0:
        return torch.zeros(t, dtype=torch.int64)
    if kind == "even":
        tok = torch.randint(1, v + 1, (t,), generator=g)
    elif kind == "hot":      # half of the tokens are one id, and some are none
        tok = torch.randint(0, v + 1, (t,), generator=g)
        tok[torch.rand(t, generator=g) < 0.5] = 1 + v // 3
    elif kind == "one":
        tok = torch.full((t,), v, dtype=torch.int64)
    else:                    # "none"
        tok = torch.zeros(t, dtype=torch.int64)
    return tok


SIZES = [(1, 1, 1), (1, 8, 5), (5, 513, 3), (31, 64, 40), (33, 7, 2), (64, 520, 1000), (256, 515, 40), (257, 72, 300), (1000, 65, 130), (1025, 16, 5000),
         (4097, 9, 70000), (5000, 1030, 11), (9000, 33, 20000)]


@pytest.mark.parametrize("ty", TYPES, ids=IDS.get)
@pytest.mark.parametrize("tw", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", [(1, 1, 1), (5, 513, 3), (64, 520, 1000), (1000, 65, 130)], ids=str)
def test_embed(size, ty, tw):
    import stade_hip
    t, d, v = size
    g = gen(t + d)
    w, tok, s = normal(g, v, d, dtype=tw), _tokens(g, t, v, "hot"), 0.375
    print(f"embed t={t} d={d} v={v} {IDS[ty]} from {IDS[tw]}", flush=True)
    y = torch.full((t, d), 5.0, dtype=ty, device="cuda")
    stade_hip.embed(y, w.cuda(), tok.cuda(), s, d, v, t, check=True)
    want = s * torch.cat([torch.zeros(1, d, dtype=torch.float64), w.double()])[tok]
    within("y", y, want, U * want.abs(), ty)
    # rows apart, at odd offsets
    yv = apart(torch.zeros(t, d, dtype=ty, device="cuda"))
    stade_hip.embed(yv, apart(w.cuda()), tok.cuda(), s, d, v, t)
    assert torch.equal(yv, y)


@pytest.mark.parametrize("tw", TYPES, ids=IDS.get)
@pytest.mark.parametrize("add", [False, True], ids=["set", "add"])
@pytest.mark.parametrize("kind", ["even", "hot", "one", "none"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_embed_b(size, kind, add, tw):
    import stade_hip
    t, d, v = size
    g = gen(t * 7 + d)
    ty = TYPES[(t + d) % 3]
    yb, tok, s = normal(g, t, d, dtype=ty), _tokens(g, t, v, kind), 0.75
    base = normal(g, v, d, dtype=tw)
    print(f"embed_b t={t} d={d} v={v} {kind} add={add} {IDS[ty]} into {IDS[tw]}", flush=True)
    wb = base.cuda() if add else torch.full((v, d), float("nan"), dtype=tw, device="cuda")
    stade_hip.embed_b(yb.cuda(), wb, tok.cuda(), s, d, v, t, add=add, check=True)
    sums = torch.zeros(v + 1, d, dtype=torch.float64).index_add_(0, tok, yb.double())[1:]
    sizes = torch.zeros(v + 1, d, dtype=torch.float64).index_add_(0, tok, yb.double().abs())[1:]
    want = s * sums + (base.double() if add else 0.0)
    # additions nest at most t deep; then the scale, and the addition to what was there
    within("wb", wb, want, U * (t * s * sizes + 2 * want.abs()), tw)
    # the same bits again, with rows apart
    again = apart(base.cuda()) if add else apart(torch.zeros(v, d, dtype=tw, device="cuda"))
    stade_hip.embed_b(apart(yb.cuda()), again, tok.cuda(), s, d, v, t, add=add)
    assert torch.equal(again, wb)


def test_embed_b_many_tokens():
    """More tokens than one block sorts, and runs over many chunks."""
    import stade_hip
    t, d, v = 70001, 24, 300000
    g = gen(3)
    yb = normal(g, t, d)
    tok = torch.where(torch.rand(t, generator=g) < 0.3, torch.full((t,), 77), torch.randint(0, v + 1, (t,), generator=g))
    print(f"embed_b t={t} d={d} v={v}", flush=True)
    wb = torch.full((v, d), float("nan"), device="cuda")
    stade_hip.embed_b(yb.cuda(), wb, tok.cuda(), 1.0, d, v, t, add=False)
    sums = torch.zeros(v + 1, d, dtype=torch.float64).index_add_(0, tok, yb.double())[1:]
    sizes = torch.zeros(v + 1, d, dtype=torch.float64).index_add_(0, tok, yb.double().abs())[1:]
    within("wb", wb, sums, U * (2100 * sizes), torch.float32)   # 32 a chunk, then 656 chunks, some 2100 at most


@pytest.mark.parametrize("size", [(1, 1), (1, 9), (63, 4), (1000, 1), (1025, 300), (4096, 5000), (16384, 70000), (16385, 70000), (40000, 3)],
                         ids=str)
def test_token_order(size):
    import stade_hip
    t, v = size
    tok = _tokens(gen(t + v), t, v, "hot")
    print(f"token_order t={t} v={v}", flush=True)
    order, start = torch.empty(t, dtype=torch.int64, device="cuda"), torch.empty(v + 1, dtype=torch.int64, device="cuda")
    stade_hip.token_order(tok.cuda(), order, start, v, t)
    key = torch.where(tok == 0, torch.full_like(tok, v), tok - 1)
    want = torch.sort(key, stable=True)
    assert torch.equal(order.cpu(), want.indices + 1)
    assert torch.equal(start.cpu(), torch.searchsorted(want.values, torch.arange(v + 1)))


def test_ids_out_of_range():
    import stade_hip
    d, v = 40, 6
    w, yb = torch.randn(v, d, device="cuda"), torch.randn(5, d, device="cuda")
    tok = torch.tensor([1, 7, -3, 2 ** 40, 6], device="cuda")
    y = torch.empty(5, d, device="cuda")
    print("embed, ids out of range", flush=True)
    with pytest.raises(stade_hip.StadeHipBoundsError):
        stade_hip.embed(y, w, tok, 1.0, d, v, 5, check=True)
    assert torch.equal(y[0], w[0]) and torch.equal(y[4], w[5]) and not y[1:4].any()
    wb = torch.empty(v, d, device="cuda")
    with pytest.raises(stade_hip.StadeHipBoundsError):
        stade_hip.embed_b(yb, wb, tok, 1.0, d, v, 5, add=False, check=True)
    assert torch.equal(wb[0], yb[0]) and torch.equal(wb[5], yb[4]) and not wb[1:5].any()
    assert stade_hip.device_error() == 0


def test_nothing():
    """No tokens, no columns, no ids."""
    import stade_hip
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    wb = torch.ones(4, 8, device="cuda")
    stade_hip.embed_b(torch.empty(0, 8, device="cuda"), wb, none, 1.0, 8, 4, 0)
    assert wb.eq(1).all()
    stade_hip.embed_b(torch.empty(0, 8, device="cuda"), wb, none, 1.0, 8, 4, 0, add=False)
    assert not wb.any()
    start = torch.ones(5, dtype=torch.int64, device="cuda")
    stade_hip.token_order(none, none, start, 4, 0)
    assert not start.any()
    y = torch.ones(3, 8, device="cuda")
    stade_hip.embed(y, torch.empty(0, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), 1.0, 8, 0, 3)
    assert not y.any()
    stade_hip.embed_b(y, torch.empty(0, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), 1.0, 8, 0, 3, add=False)


def test_gradient_by_differences():
    """embed is linear in w: <yb, embed(w + v) - embed(w - v)> / 2 = <wb, v>."""
    import stade_hip
    t, d, v = 300, 33, 50
    g = gen(9)
    w, dv, yb = (cuda(normal(g, *s)) for s in ((v, d), (v, d), (t, d)))
    tok = _tokens(g, t, v, "hot").cuda()
    ys = []
    for sign in (1, -1):
        y = torch.empty(t, d, device="cuda")
        stade_hip.embed(y, w + sign * dv, tok, 0.5, d, v, t)
        ys.append(y.double())
    wb = torch.zeros(v, d, device="cuda")
    stade_hip.embed_b(yb, wb, tok, 0.5, d, v, t)
    left = (yb.double() * (ys[0] - ys[1])).sum() / 2
    right = (wb.double() * dv.double()).sum()
    # the inputs w +- v and the outputs are each rounded once; wb's sums nest t deep
    slack = U * (2 * (yb.double() * (ys[0].abs() + ys[1].abs())).abs().sum() + t * (yb.double().abs().sum(0).max() * dv.double().abs().sum()))
    assert abs(left - right) <= slack
