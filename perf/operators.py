"""Performance cases of the language-model operators: token rows, layer norm, the 8-bit tape
and products by expert, each in its plain form and through the framework's entry points.

A case is one use of one operator ("kind") at one size and type.  Arrays are row by row (the
entry points' column-major (i_d, i_n) array is a torch tensor (n, d)); tokens count from 1 and
0 is "no token".  Where `own` is false `run` computes the plain form in 32 bits and rounds once
at the end; where it is true it calls the framework.  `exact` gives the same in 64 bits."""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
GROUP = 32        # values of a row that share a tape scale
EPS = 1e-5
EMBED_SCALE = 8.0


def listed():
    return [
        # a decoding step's token rows: one short launch
        {"name": "embed_16x1024", "kind": "embed", "t": 16, "d": 1024, "v": 32768, "type": "bf16"},
        # a training step's embedding gradient: frequent and rare tokens, a large table
        {"name": "embed_b_16384x2048", "kind": "embed_b", "t": 16384, "d": 2048, "v": 65536, "type": "bf16", "grad": "f32"},
        # the same of a small model with odd sizes
        {"name": "embed_b_3001x515", "kind": "embed_b", "t": 3001, "d": 515, "v": 10007, "type": "f32", "grad": "f32"},
        # tokens sent to their experts: the order by expert, and the rows taken in that order
        {"name": "route_5000x1111", "kind": "route", "t": 5000, "d": 1111, "v": 60, "type": "f16"},
        # a decoding step's layer norm: one short launch
        {"name": "norm_8x1024", "kind": "norm", "n": 8, "d": 1024, "type": "bf16"},
        # the reverse sweep of a training step's layer norm, with its weights' gradients
        {"name": "norm_b_16384x4096", "kind": "norm_b", "n": 16384, "d": 4096, "type": "bf16"},
        # both sweeps in 32 bits at odd sizes
        {"name": "norm_both_2999x777", "kind": "norm_both", "n": 2999, "d": 777, "type": "f32"},
        # both sweeps with the input held in 8 bits between them
        {"name": "norm_tape_8192x4096", "kind": "norm_tape", "n": 8192, "d": 4096, "type": "bf16"},
        # products of a training batch's tokens with their experts' weights
        {"name": "expert_8192", "kind": "expert", "t": 8192, "i": 2048, "o": 4096, "e": 8, "skew": 0.3, "type": "bf16"},
        # a decoding step's tokens: a few rows an expert, bound by reading the weights
        {"name": "expert_24", "kind": "expert", "t": 24, "i": 2048, "o": 4096, "e": 8, "skew": 0.3, "type": "bf16"},
        # the reverse sweep, the rows held in 8 bits for the weights' gradient
        {"name": "expert_b_tape_16384", "kind": "expert_b_tape", "t": 16384, "i": 2048, "o": 4096, "e": 16, "skew": 0.3,
         "type": "bf16", "grad": "f32"},
        # both sweeps of a small model: sizes that fill no tile, some experts with few rows
        {"name": "expert_both_1000", "kind": "expert_both", "t": 1000, "i": 500, "o": 700, "e": 7, "skew": 1.0, "type": "f16",
         "grad": "f32"},
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _size(rng, lo, hi, step):
    """As `_between`; half of the time the nearest multiple of `step`, as users often choose."""
    v = _between(rng, lo, hi)
    return max(step, v // step * step) if rng.random() < 1 / 2 else v


def draw(rng):
    kind = rng.choice(("embed", "embed_b", "route", "norm", "norm_b", "norm_both", "norm_tape", "tape", "expert", "expert_b",
                       "expert_b_tape", "expert_both"))
    c = {"kind": kind, "type": rng.choice(("bf16", "bf16", "f16", "f32"))}
    if kind in ("embed", "embed_b", "route"):
        c.update(t=_size(rng, 1, 16384, 64), d=_size(rng, 64, 4096, 64))
        c["v"] = _between(rng, 4, 256) if kind == "route" else min(_between(rng, 500, 131072), (1 << 27) // c["d"])
    elif kind.startswith("norm") or kind == "tape":
        c["d"] = _size(rng, 64, 8192, 64)
        c["n"] = _size(rng, 1, min(16384, (1 << 26) // c["d"]), 64)
    else:
        c.update(t=_size(rng, 1, 8192, 64), i=_size(rng, 128, 2048, 64), o=_size(rng, 128, 4096, 64), e=rng.choice((2, 4, 8, 16, 32)),
                 skew=round(rng.uniform(0.0, 1.0), 2))
    if kind == "embed_b" or kind.startswith("expert_b"):
        c["grad"] = rng.choice(("f32", c["type"]))
    return c


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _tokens(g, t, v):
    """Ids 1..v with frequencies that fall like a power of their rank, ranks spread over the
    ids, and one in fifty 0 (padding)."""
    u = torch.rand(t, generator=g, device=DEV, dtype=torch.float64)
    rank = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
    step = next(p for p in (7919, 7907, 7901, 7883) if v % p)
    tok = (rank * step) % v + 1
    return torch.where(torch.rand(t, generator=g, device=DEV) < 0.02, torch.zeros_like(tok), tok)


def _starts(g, t, e, skew):
    """Row offsets of e experts with uneven shares of t rows."""
    share = torch.exp(skew * torch.randn(e, generator=g, device=DEV, dtype=torch.float64))
    cut = torch.round(torch.cumsum(share, 0) / share.sum() * t).long()
    cut[-1] = t
    return torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), cut])


def _inputs(case, seed):
    g, kind, dt = _gen(seed), case["kind"], TYPES[case["type"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    if kind in ("embed", "embed_b"):
        t, d, v = case["t"], case["d"], case["v"]
        s = {"tok": _tokens(g, t, v)}
        s["w" if kind == "embed" else "yb"] = normal(v, d, scale=0.02) if kind == "embed" else normal(t, d)
        return s
    if kind == "route":
        ids = torch.randint(1, case["v"] + 1, (case["t"],), generator=g, device=DEV)
        return {"tok": ids, "w": normal(case["t"], case["d"])}
    if kind.startswith("norm"):
        n, d = case["n"], case["d"]
        # rows of different sizes, as a residual stream has them, a few columns much larger
        x = torch.randn(n, d, generator=g, device=DEV) * torch.exp(0.5 * torch.randn(n, 1, generator=g, device=DEV)) + 0.3
        x[:, :: max(1, d // 5)] *= 6.0
        s = {"x": x.to(dt), "g": 1.0 + 0.1 * torch.randn(d, generator=g, device=DEV), "b": 0.1 * torch.randn(d, generator=g, device=DEV)}
        if kind != "norm":
            s["yb"] = normal(n, d)
        if kind == "norm_b":   # what the forward sweep left
            xf = s["x"].float()
            s["mu"] = xf.mean(1)
            s["rs"] = torch.rsqrt(xf.sub(s["mu"][:, None]).square().mean(1) + EPS)
        return s
    if kind == "tape":
        return {"x": normal(case["n"], case["d"]) * torch.exp(normal(case["n"], 1)).to(dt)}
    t, i, o, e = case["t"], case["i"], case["o"], case["e"]
    s = {"x": normal(t, i), "w": normal(e, i, o, scale=1.0 / math.sqrt(i)), "start": _starts(g, t, e, case["skew"])}
    if kind != "expert":
        s["yb"] = normal(t, o)
    return s


def prepare(case, seed):
    """The inputs, and the arrays that a program keeps for the results."""
    s, kind, dt = _inputs(case, seed), case["kind"], TYPES[case["type"]]

    def new(*shape, dtype=dt):
        return torch.empty(*shape, dtype=dtype, device=DEV)

    if kind == "embed":
        s["y"] = new(case["t"], case["d"])
    elif kind == "embed_b":
        s["wb"] = new(case["v"], case["d"], dtype=TYPES[case["grad"]])
    elif kind == "route":
        s.update(order=new(case["t"], dtype=torch.int64), start=new(case["v"] + 1, dtype=torch.int64), y=new(case["t"], case["d"]))
    elif kind.startswith("norm"):
        n, d = case["n"], case["d"]
        if kind != "norm_b":
            s.update(y=new(n, d), mu=new(n, dtype=torch.float32), rs=new(n, dtype=torch.float32))
        if kind != "norm":
            s.update(xb=new(n, d), gb=new(d, dtype=torch.float32), bb=new(d, dtype=torch.float32))
    elif kind == "tape":
        s["back"] = new(case["n"], case["d"])
    else:
        t, i, o, e = case["t"], case["i"], case["o"], case["e"]
        if kind in ("expert", "expert_both"):
            s["y"] = new(t, o)
        if kind != "expert":
            s.update(xb=new(t, i), wb=new(e, i, o, dtype=TYPES[case["grad"]]))
        # the longest expert's rows, for the plain form's padded products
        s["longest"] = int((s["start"][1:] - s["start"][:-1]).max())
    if kind in ("norm_tape", "tape", "expert_b_tape"):
        n, d = (case["t"], case["i"]) if kind == "expert_b_tape" else (case["n"], case["d"])
        groups = -(-d // GROUP)
        s.update(q=new(n, groups * GROUP, dtype=torch.int8), qs=new(n, groups, dtype=torch.uint8))
    return case, s


# ------------------------------------------------------------------------------------------
# the plain forms, in 32 bits
# ------------------------------------------------------------------------------------------

def _tape_values(x):
    """The values that the 8-bit tape of x holds: a power-of-two scale for each 32 of a row, the
    least one with |x| / scale <= 127, and whole numbers of it."""
    n, d = x.shape
    v = torch.nn.functional.pad(x, (0, -d % GROUP)).view(n, -1, GROUP)
    m, k = torch.frexp(v.abs().amax(2, keepdim=True))          # amax = m 2^k, 1/2 <= m < 1
    up = torch.ldexp(torch.ones_like(m), torch.clamp(k - 7 + (m > 127 / 128), min=-126))
    return (torch.round(v / up) * up).view(n, -1)[:, :d]


def _norm(x, g, b):
    mu = x.mean(1, keepdim=True)
    c = x - mu
    rs = torch.rsqrt((c * c).mean(1, keepdim=True) + EPS)
    return c * rs * g + b, mu, rs


def _norm_b(yb, x, g, mu, rs):
    xh = (x - mu) * rs
    a = yb * g
    xb = rs * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    return xb, (yb * xh).sum(0), yb.sum(0)


def _places(s, t, e):
    """Each row's expert and its place among that expert's rows."""
    row = torch.arange(t, device=DEV)
    ex = torch.searchsorted(s["start"][1:], row, right=True)
    return ex, row - s["start"][ex]


def _padded(v, ex, at, e, longest):
    p = torch.zeros(e, longest, v.shape[1], dtype=torch.float32, device=DEV)
    p[ex, at] = v.float()
    return p


def _plain(case, s):
    kind, dt = case["kind"], TYPES[case["type"]]
    if kind == "embed":
        y = s["w"][(s["tok"] - 1).clamp_min(0)].float()
        return {"y": (y * EMBED_SCALE * (s["tok"] > 0)[:, None]).to(dt)}
    if kind == "embed_b":
        wb = torch.zeros(case["v"] + 1, case["d"], dtype=torch.float32, device=DEV)
        wb.index_add_(0, s["tok"], s["yb"].float() * EMBED_SCALE)
        return {"wb": wb[1:].to(TYPES[case["grad"]])}
    if kind == "route":
        order = torch.sort(s["tok"], stable=True).indices
        start = torch.cumsum(torch.bincount(s["tok"], minlength=case["v"] + 1), 0)
        return {"order": order + 1, "start": start, "y": s["w"][order]}
    if kind.startswith("norm"):
        out = {}
        x, g, b = s["x"].float(), s["g"], s["b"]
        mu, rs = (s["mu"][:, None], s["rs"][:, None]) if kind == "norm_b" else (None, None)
        if kind != "norm_b":
            y, mu, rs = _norm(x, g, b)
            out.update(y=y.to(dt), mu=mu[:, 0], rs=rs[:, 0])
        if kind != "norm":
            xb, gb, bb = _norm_b(s["yb"].float(), _tape_values(x) if kind == "norm_tape" else x, g, mu, rs)
            out.update(xb=xb.to(dt), gb=gb, bb=bb)
        return out
    if kind == "tape":
        return {"back": _tape_values(s["x"].float()).to(dt)}
    e, out = case["e"], {}
    ex, at = _places(s, case["t"], e)
    w = s["w"].float()
    if kind in ("expert", "expert_both"):
        out["y"] = torch.bmm(_padded(s["x"], ex, at, e, s["longest"]), w)[ex, at].to(dt)
    if kind != "expert":
        yb = _padded(s["yb"], ex, at, e, s["longest"])
        x = _tape_values(s["x"].float()) if kind == "expert_b_tape" else s["x"]
        out["xb"] = torch.bmm(yb, w.transpose(1, 2).contiguous())[ex, at].to(dt)
        out["wb"] = torch.bmm(_padded(x, ex, at, e, s["longest"]).transpose(1, 2).contiguous(), yb).to(TYPES[case["grad"]])
    return out


# ------------------------------------------------------------------------------------------
# the framework's operators
# ------------------------------------------------------------------------------------------

_lib = []


def _hip():
    if not _lib:
        pkg = str(Path.cwd() / "stade.jl_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import stade_hip
        _lib.append(stade_hip)
    return _lib[0]


def _own(case, s):
    hip, kind = _hip(), case["kind"]
    if kind == "embed":
        hip.embed(s["y"], s["w"], s["tok"], EMBED_SCALE, case["d"], case["v"], case["t"])
        return {"y": s["y"]}
    if kind == "embed_b":
        hip.embed_b(s["yb"], s["wb"], s["tok"], EMBED_SCALE, case["d"], case["v"], case["t"], add=False)
        return {"wb": s["wb"]}
    if kind == "route":
        hip.token_order(s["tok"], s["order"], s["start"], case["v"], case["t"])
        hip.embed(s["y"], s["w"], s["order"], 1.0, case["d"], case["t"], case["t"])
        return {"order": s["order"], "start": s["start"], "y": s["y"]}
    tape = (s["q"], s["qs"]) if "q" in s else None
    if kind.startswith("norm"):
        n, d = case["n"], case["d"]
        if kind != "norm_b":
            hip.layernorm(s["y"], s["x"], s["g"], s["b"], s["mu"], s["rs"], d, n, eps=EPS, tape=tape)
        if kind != "norm":
            hip.layernorm_b(s["yb"], None if tape else s["x"], s["xb"], s["g"], s["gb"], s["bb"], s["mu"], s["rs"], d, n, add=False,
                            tape=tape)
        names = {"norm": ("y", "mu", "rs"), "norm_b": ("xb", "gb", "bb")}.get(kind, ("y", "mu", "rs", "xb", "gb", "bb"))
        return {a: s[a] for a in names}
    if kind == "tape":
        hip.tape8_store(s["x"], s["q"], s["qs"], case["d"], case["n"])
        hip.tape8_load(s["q"], s["qs"], s["back"], case["d"], case["n"])
        return {"back": s["back"]}
    size, out = (case["i"], case["o"], case["t"], case["e"]), {}
    if kind in ("expert", "expert_both"):
        hip.expert_mul(s["y"], s["x"], s["w"], s["start"], *size)
        out["y"] = s["y"]
    if kind == "expert_b_tape":
        hip.tape8_store(s["x"], s["q"], s["qs"], case["i"], case["t"])
    if kind != "expert":
        hip.expert_mul_b(s["yb"], None if tape else s["x"], s["xb"], s["w"], s["wb"], s["start"], *size, add=False, tape=tape)
        out.update(xb=s["xb"], wb=s["wb"])
    return out


def run(state):
    return _own(*state) if own else _plain(*state)


# ------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------

def work(case):
    kind, b = case["kind"], TYPES[case["type"]].itemsize
    if kind == "embed":
        t, d = case["t"], case["d"]
        return {"bytes": float(t * (8 + 2 * d * b)), "flops": float(t * d)}
    if kind == "embed_b":
        t, d = case["t"], case["d"]
        return {"bytes": float(t * (8 + d * b) + case["v"] * d * TYPES[case["grad"]].itemsize), "flops": float(2 * t * d)}
    if kind == "route":
        t, d = case["t"], case["d"]
        return {"bytes": float(t * (16 + 2 * d * b) + 8 * (case["v"] + 1)), "flops": 0.0}
    if kind == "tape":   # the values in, the tape out, the tape in, the values out
        nd = case["n"] * case["d"]
        return {"bytes": float(nd * (2 * b + 2) + 2 * case["n"] * -(-case["d"] // GROUP)), "flops": float(3 * nd)}
    if kind.startswith("norm"):
        nd, n, d = case["n"] * case["d"], case["n"], case["d"]
        fwd, bwd = kind != "norm_b", kind != "norm"
        size = (2 * nd * b + 8 * n + 8 * d) * fwd + (3 * nd * b + 8 * n + 12 * d) * bwd
        if kind == "norm_tape":   # 8 bits and a 32nd written, and read in place of x
            size += 2 * nd + 2 * n * -(-d // GROUP) - nd * b
        return {"bytes": float(size), "flops": float(nd * (8 * fwd + 14 * bwd))}
    t, i, o, e = case["t"], case["i"], case["o"], case["e"]
    e = min(e, t)   # experts with rows
    fwd, bwd = kind in ("expert", "expert_both"), kind != "expert"
    size = (t * (i + o) * b + e * i * o * b) * fwd
    if bwd:
        size += t * (2 * i + o) * b + e * i * o * (b + TYPES[case["grad"]].itemsize)
    if kind == "expert_b_tape":   # x read once to be stored, the tape written and read
        size += 2 * t * i + 2 * t * -(-i // GROUP)
    return {"bytes": float(size), "flops": 2.0 * t * i * o * (fwd + 2 * bwd)}


# ------------------------------------------------------------------------------------------
# the same in 64 bits
# ------------------------------------------------------------------------------------------

def _exact_tape(x):
    out = torch.zeros_like(x)
    for j in range(0, x.shape[1], GROUP):
        part = x[:, j:j + GROUP]
        big = part.abs().amax(1)
        e = torch.where(big > 0, torch.ceil(torch.log2(big / 127.0)), torch.full_like(big, -126.0))
        # the least e with big <= 127 * 2^e, whatever the logarithm's rounding
        e = torch.where(big <= 127.0 * torch.exp2(e - 1), e - 1, e)
        e = torch.where(big > 127.0 * torch.exp2(e), e + 1, e).clamp_min(-126.0)
        unit = torch.exp2(e)[:, None]
        out[:, j:j + GROUP] = torch.round(part / unit) * unit
    return out


def exact(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    f = {k: v.double() if v.is_floating_point() else v for k, v in s.items()}
    if kind == "embed":
        table = torch.cat([torch.zeros(1, case["d"], dtype=torch.float64, device=DEV), f["w"]])
        return {"y": EMBED_SCALE * table.index_select(0, s["tok"])}
    if kind == "embed_b":
        wb = torch.zeros(case["v"] + 1, case["d"], dtype=torch.float64, device=DEV)
        wb.index_put_((s["tok"],), f["yb"], accumulate=True)
        return {"wb": EMBED_SCALE * wb[1:]}
    if kind == "route":
        t = case["t"]
        order = torch.argsort(s["tok"] * t + torch.arange(t, device=DEV))
        start = torch.searchsorted(s["tok"][order], torch.arange(1, case["v"] + 2, device=DEV))
        return {"order": order + 1, "start": start, "y": f["w"].index_select(0, order)}
    if kind.startswith("norm"):
        n, d, x, out = case["n"], case["d"], f["x"], {}
        if kind == "norm_b":   # of the statistics that it is given
            mu, rs = f["mu"], f["rs"]
        else:
            mu = x.sum(1) / d
            rs = 1.0 / torch.sqrt(((x - mu[:, None]) ** 2).sum(1) / d + EPS)
            out = {"y": (x - mu[:, None]) * rs[:, None] * f["g"] + f["b"], "mu": mu, "rs": rs}
        if kind != "norm":
            held = _exact_tape(x) if kind == "norm_tape" else x
            xh = (held - mu[:, None]) * rs[:, None]
            a = f["yb"] * f["g"]
            out["xb"] = rs[:, None] * (a - a.sum(1)[:, None] / d - xh * ((a * xh).sum(1) / d)[:, None])
            out["gb"] = (f["yb"] * xh).sum(0)
            out["bb"] = f["yb"].sum(0)
        return out
    if kind == "tape":
        return {"back": _exact_tape(f["x"])}
    t, i, o, e = case["t"], case["i"], case["o"], case["e"]
    cut, out = s["start"].tolist(), {}
    held = _exact_tape(f["x"]) if kind == "expert_b_tape" else f["x"]
    y = torch.zeros(t, o, dtype=torch.float64, device=DEV)
    xb = torch.zeros(t, i, dtype=torch.float64, device=DEV)
    wb = torch.zeros(e, i, o, dtype=torch.float64, device=DEV)
    for k in range(e):
        rows = slice(cut[k], cut[k + 1])
        if cut[k] == cut[k + 1]:
            continue
        if kind in ("expert", "expert_both"):
            y[rows] = f["x"][rows].mm(f["w"][k])
        if kind != "expert":
            xb[rows] = f["yb"][rows].mm(f["w"][k].t().contiguous())
            wb[k] = held[rows].t().contiguous().mm(f["yb"][rows])
    if kind in ("expert", "expert_both"):
        out["y"] = y
    if kind != "expert":
        out.update(xb=xb, wb=wb)
    return out
