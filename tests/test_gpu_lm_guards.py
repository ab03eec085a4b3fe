"""What the language-model operators leave alone: the elements before an output, between its rows
and behind it, at lengths that end inside a vector, a group or a tile."""
import pytest
import torch

from lmhelp import IDS, TYPES, gen, normal

pytestmark = pytest.mark.gpu


class Guarded:
    """An output of n rows of d, `gap` elements apart, in a buffer whose other elements must not change."""

    def __init__(self, n, d, dtype, gap=0, lead=64):
        self.buf = torch.empty(lead + n * (d + gap) + 64, dtype=dtype, device="cuda").fill_(77)
        self.view = self.buf[lead:lead + n * (d + gap)].view(n, d + gap)[:, :d]
        self.out = torch.ones_like(self.buf, dtype=torch.bool)
        self.out[lead:lead + n * (d + gap)].view(n, d + gap)[:, :d] = False

    def vector(self):
        return self.view[0]

    def check(self, name):
        bad = (self.buf != 77) & self.out
        assert not bad.any(), f"{name}: written at {bad.nonzero().flatten()[:8].tolist()}"


class Outputs(dict):
    def add(self, name, n, d, dtype, gap=0, lead=64):
        self[name] = Guarded(n, d, dtype, gap, lead)
        return self[name].view

    def vec(self, name, n, dtype):
        self.add(name, 1, n, dtype)
        return self[name].vector()

    def tape(self, d, n):
        g = -(-d // 32)
        return self.vec("q", 32 * g * n, torch.int8), self.vec("qs", g * n, torch.uint8)

    def check(self):
        torch.cuda.synchronize()
        for name, g in self.items():
            g.check(name)


# (gap between rows, elements before the first): packed, and apart at an odd offset
PLACES = [(0, 64), (3, 65)]


@pytest.mark.parametrize("place", PLACES, ids=["packed", "apart"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("d", [1, 5, 9, 33, 127, 129, 513, 515, 1027, 2050, 4099, 8201, 16387, 33001])
def test_norm_and_tape(d, dt, place):
    import stade_hip as hip
    n, o = (7 if d < 8000 else 3), Outputs()
    g = gen(d)
    x, yb = normal(g, n, d, dtype=dt).cuda(), normal(g, n, d, dtype=dt).cuda()
    w = torch.ones(d, device="cuda")
    f32 = torch.float32
    print(f"guards: layernorm, tape8 d={d} {IDS[dt]} {place}", flush=True)
    tape = o.tape(d, n)
    hip.layernorm(o.add("y", n, d, dt, *place), x, w, w, o.vec("mu", n, f32), o.vec("rs", n, f32), d, n, tape=tape)
    mu, rs = o["mu"].vector(), o["rs"].vector()
    o.check()
    for add in (False, True):
        hip.layernorm_b(yb, x, o.add("xb", n, d, dt, *place), w, o.vec("gb", d, f32), o.vec("bb", d, f32), mu, rs, d, n, add=add)
        o.check()
        hip.layernorm_b(yb, None, o.add("xb", n, d, dt, *place), w, o.vec("gb", d, f32), o.vec("bb", d, f32), mu, rs, d, n, add=add, tape=tape)
        o.check()
    # more rows than one block takes
    many = 70
    xs, ys = x.repeat(many // n + 1, 1)[:many], yb.repeat(many // n + 1, 1)[:many]
    hip.layernorm_b(ys, xs, o.add("xb", many, d, dt, *place), w, o.vec("gb", d, f32), o.vec("bb", d, f32), mu.repeat(many)[:many].contiguous(),
                    rs.repeat(many)[:many].contiguous(), d, many, add=False)
    o.check()
    tape = o.tape(d, n)
    hip.tape8_store(x, *tape, d, n)
    hip.tape8_load(*tape, o.add("back", n, d, dt, *place), d, n)
    o.check()


@pytest.mark.parametrize("place", PLACES, ids=["packed", "apart"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", [(3, 5, 4), (70, 513, 9), (250, 33, 400), (300, 7, 50), (1000, 519, 700), (9000, 35, 900), (20000, 11, 3000)], ids=str)
def test_embed(size, dt, place):
    import stade_hip as hip
    (t, d, v), o = size, Outputs()
    g = gen(t)
    w, yb = normal(g, v, d, dtype=dt).cuda(), normal(g, t, d, dtype=dt).cuda()
    tok = torch.randint(0, v + 1, (t,), generator=g)
    tok[: t // 3] = v   # (the last row too, and a run over many chunks)
    tok = tok.cuda()
    print(f"guards: embed t={t} d={d} v={v} {IDS[dt]} {place}", flush=True)
    hip.embed(o.add("y", t, d, dt, *place), w, tok, 0.5, d, v, t)
    for add in (False, True):
        hip.embed_b(yb, o.add("wb", v, d, dt, *place), tok, 0.5, d, v, t, add=add)
        o.check()
    hip.embed_b(yb[:0], o.add("wb", v, d, dt, *place), tok[:0], 0.5, d, v, 0, add=False)
    hip.token_order(tok, o.vec("order", t, torch.int64), o.vec("start", v + 1, torch.int64), v, t)
    o.check()


# (small tiles, k in slices, tiles of 128 x 128 and of 256 x 256 of 16-bit values; straight and through registers)
@pytest.mark.parametrize("place", PLACES + [(8, 64)], ids=["packed", "apart", "apart, aligned"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", [([3, 0, 5], 2, 33, 41), ([70, 65], 1, 72, 200), ([40], 0, 64, 2104), ([20, 0, 31], 0, 2001, 71), ([900, 0, 301], 3, 64, 4104),
                                  ([900, 0, 301], 3, 4104, 72), ([5] * 130, 3, 300, 260), ([700, 515], 0, 67, 16387)],
                         ids=lambda s: f"{len(s[0])}x{sum(s[0])}+{s[1]}-{s[2]}-{s[3]}")
def test_expert_mul(size, dt, place):
    import stade_hip as hip
    (counts, rest, i, o_), o = size, Outputs()
    t, e = sum(counts) + rest, len(counts)
    g = gen(t + i)
    x, w, yb = (normal(g, *s, dtype=dt).cuda() for s in ((t, i), (e, i, o_), (t, o_)))
    start = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist()).cuda()
    tape = Outputs().tape(i, t)
    hip.tape8_store(x, *tape, i, t)
    print(f"guards: expert_mul {size} {IDS[dt]} {place}", flush=True)
    for add in (False, True):
        hip.expert_mul(o.add("y", t, o_, dt, *place), x, w, start, i, o_, t, e, add=add)
        o.check()
        for grad in {dt, torch.float32}:
            wb = o.vec("wb", e * i * o_, grad)
            hip.expert_mul_b(yb, x, o.add("xb", t, i, dt, *place), w, wb, start, i, o_, t, e, add=add)
            o.check()
            wb = o.vec("wb", e * i * o_, grad)
            hip.expert_mul_b(yb, None, None, None, wb, start, i, o_, t, e, add=add, tape=tape)
            o.check()
