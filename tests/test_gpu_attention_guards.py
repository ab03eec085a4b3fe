"""What the operators around attention and the experts leave alone: the elements before an output, between its rows and
behind it."""
import pytest
import torch

from lmhelp import IDS, TYPES, gen, normal
from test_gpu_lm_guards import PLACES, Outputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("place", PLACES, ids=["packed", "apart"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", [(1, 1, 1), (37, 2, 1), (300, 6, 2), (129, 1, 1)], ids=str)
@pytest.mark.parametrize("d", [1, 8, 20, 64, 72, 97, 128])
def test_attention(d, size, dt, place):
    import stade_hip as hip
    (t, hq, hk), o = size, Outputs()
    g = gen(d + t)
    q, yb = normal(g, t, hq * d, dtype=dt).cuda(), normal(g, t, hq * d, dtype=dt).cuda()
    k, v = normal(g, t + 5, hk * d, dtype=dt).cuda(), normal(g, t + 5, hk * d, dtype=dt).cuda()
    qs, ks = torch.tensor([0, t // 2, t]).cuda(), torch.tensor([0, t // 2 + 2, t + 3]).cuda()
    print(f"guards: attention d={d} {size} {IDS[dt]} {place}", flush=True)
    y, lse = o.add("y", t, hq * d, dt, *place), o.vec("lse", t * hq, torch.float32).view(t, hq)
    hip.attention(y, lse, q, k, v, qs, ks, 0.3, d, hq, hk, t, t + 5, 2, window=60, sinks=2)
    o.check()
    yc = y.contiguous()
    for add in (False, True):
        qb, kb, vb = o.add("qb", t, hq * d, dt, *place), o.add("kb", t + 5, hk * d, dt, *place), o.add("vb", t + 5, hk * d, dt, *place)
        hip.attention_b(yb, yc, lse, q, qb, k, kb, v, vb, qs, ks, 0.3, d, hq, hk, t, t + 5, 2, window=60, sinks=2, add=add)
        o.check()


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("d", [1, 33, 64, 128])
def test_attention_split(d, dt):
    """Keys over several blocks."""
    import stade_hip as hip
    o, g, tk = Outputs(), gen(d), 4000
    q, k, v = normal(g, 3, 4 * d, dtype=dt).cuda(), normal(g, tk, 2 * d, dtype=dt).cuda(), normal(g, tk, 2 * d, dtype=dt).cuda()
    qs, ks = torch.tensor([0, 1, 2]).cuda(), torch.tensor([0, 3000, tk]).cuda()
    print(f"guards: attention over blocks d={d} {IDS[dt]}", flush=True)
    hip.attention(o.add("y", 3, 4 * d, dt, 3, 65), o.vec("lse", 12, torch.float32).view(3, 4), q, k, v, qs, ks, 0.3, d, 4, 2, 3, tk, 2)
    o.check()
    assert not o["y"].view[2].any()     # (a column of no sequence)


@pytest.mark.parametrize("place", PLACES, ids=["packed", "apart"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("form", [(1, 0), (2, 2), (20, 6), (64, 64), (72, 30), (130, 128), (256, 256)], ids=str)
def test_head_rotary(form, dt, place):
    import stade_hip as hip
    (d, r), o = form, Outputs()
    for t, hq, hk in ((1, 2, 1), (301, 3, 2), (40, 0, 3)):
        g, width = gen(d + t), d * (hq + hk)
        x, yb = normal(g, t, width, dtype=dt).cuda(), normal(g, t, width, dtype=dt).cuda()
        gq = torch.ones(d, device="cuda")
        pos, freq = torch.arange(t).cuda(), torch.from_numpy(hip.rotary_freq(r)).cuda()
        print(f"guards: head_rotary {form} {t} {IDS[dt]} {place}", flush=True)
        for half in (True, False):
            hip.head_rotary(o.add("y", t, width, dt, *place), x, gq, gq, pos, freq, d, hq, hk, r, t, half=half)
            for add in (False, True):
                hip.head_rotary_b(yb, x, o.add("xb", t, width, dt, *place), gq, o.vec("gqb", d, torch.float32), gq, o.vec("gkb", d, torch.float32), pos, freq,
                                  d, hq, hk, r, t, half=half, add=add)
            o.check()


@pytest.mark.parametrize("place", PLACES, ids=["packed", "apart"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("d", [1, 7, 8, 513, 1025, 4099])
def test_expert_rows_and_dropout(d, dt, place):
    import stade_hip as hip
    o, g = Outputs(), gen(d)
    i64, f32 = torch.int64, torch.float32
    for t, k, e in ((1, 1, 1), (37, 3, 5), (1100, 2, 40)):
        ids = torch.randint(0, e + 1, (t, k), generator=g).cuda()
        print(f"guards: expert rows, dropout d={d} {t} {IDS[dt]} {place}", flush=True)
        order, at, start = o.vec("order", t * k, i64), o.vec("place", t * k, i64).view(t, k), o.vec("start", e + 1, i64)
        hip.expert_order(ids, order, at, start, k, e, t, check=True)
        o.check()
        x, ys, p = normal(g, t, d, dtype=dt).cuda(), normal(g, t * k, d, dtype=dt).cuda(), torch.rand(t, k, device="cuda")
        xs = o.add("xs", t * k, d, dt, *place)
        hip.expert_take(xs, x, at, d, k, t, check=True)
        used = int(start[-1])
        assert (xs[used:] == 77).all()      # (columns that no place names)
        for add in (False, True):
            hip.expert_take_b(ys, o.add("xb", t, d, dt, *place), at, d, k, t, add=add)
            hip.expert_join(o.add("y", t, d, dt, *place), ys, p, at, d, k, t, add=add)
            ysb = o.add("ysb", t * k, d, dt, *place)
            hip.expert_join_b(x, ys, ysb, p, o.vec("pb", t * k, f32).view(t, k), at, d, k, t, add=add)
            assert (ysb[used:] == 77).all()
        key = torch.tensor([3, 4]).cuda()
        hip.dropout(o.add("dropped", t, d, dt, *place), x, x, key, 0.3, d, t)
        hip.dropout_b(x, o.add("droppedb", t, d, dt, *place), key, 0.3, d, t, add=False)
        o.check()
