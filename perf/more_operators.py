"""Performance cases of the operators around attention and the experts: positions of queries and
keys (`head_rotary`), attention over ragged sequences (`attention`), tokens sent to several experts and
back (`expert_order`, `expert_take`, `expert_join`) and dropout without a stored mask (`dropout`), each in
its plain form and through the framework's entry points.

A case is one use of one operator ("kind") at one size and type.  Arrays are row by row (the entry
points' column-major (i_d, i_n) array is a torch tensor (n, d)).  Places count from 1 and 0 is "none"; offsets of
sequences and positions count from 0.  Where `own` is false `run` computes the plain form in 32 bits and
rounds once at the end; where it is true it calls the framework.  `exact` gives the same in 64 bits."""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
BASE = 10000.0
DROP = 0.1


def listed():
    return [
        # a decoding step's queries and keys, normed and rotated: one short launch
        {"name": "rotary_16x40x128", "kind": "rotary", "t": 16, "hq": 32, "hk": 8, "d": 128, "r": 128, "half": True, "norm": True, "far": 100000,
         "type": "bf16"},
        # a training step's, both sweeps with the norms' weights, a part of each head rotated by neighbouring pairs
        {"name": "rotary_both_8192x20x128", "kind": "rotary_both", "t": 8192, "hq": 16, "hk": 4, "d": 128, "r": 64, "half": False, "norm": True,
         "far": 0, "type": "bf16"},
        # one user's decoding step after a short prompt: latency
        {"name": "attn_1x500", "kind": "attn", "n": 1, "t": 1, "tk": 500, "hq": 16, "hk": 4, "d": 64, "w": 1024, "sinks": 4, "type": "f16"},
        # a batch's decoding step over long and short contexts: bound by reading the keys and values
        {"name": "attn_64x4096", "kind": "attn", "n": 64, "t": 64, "tk": 262144, "hq": 32, "hk": 8, "d": 128, "w": 8192, "sinks": 4, "type": "bf16"},
        # chunks of new tokens behind long contexts, all of them visible
        {"name": "attn_chunk_4x512", "kind": "attn", "n": 4, "t": 2048, "tk": 34816, "hq": 16, "hk": 4, "d": 128, "w": -1, "sinks": 0, "type": "bf16"},
        # prompts of uneven lengths under a window and sinks
        {"name": "attn_5x3300", "kind": "attn", "n": 5, "t": 16500, "tk": 16500, "hq": 32, "hk": 8, "d": 128, "w": 1024, "sinks": 4, "type": "bf16"},
        # a training step's attention, both sweeps
        {"name": "attn_both_4x2048", "kind": "attn_both", "n": 4, "t": 8192, "tk": 8192, "hq": 16, "hk": 4, "d": 128, "w": 1024, "sinks": 4,
         "type": "bf16"},
        # the same of a small model in 32 bits at odd sizes
        {"name": "attn_both_3x500", "kind": "attn_both", "n": 3, "t": 1501, "tk": 1501, "hq": 6, "hk": 2, "d": 80, "w": 300, "sinks": 1, "type": "f32"},
        # a training step's tokens sent to two experts each and back, both sweeps
        {"name": "moe_both_8192x2048", "kind": "moe_both", "t": 8192, "k": 2, "e": 64, "d": 2048, "type": "bf16"},
        # a small batch at an odd width
        {"name": "moe_77x1111", "kind": "moe", "t": 77, "k": 4, "e": 30, "d": 1111, "type": "f32"},
        # dropout on a residual branch of a training step, both sweeps
        {"name": "drop_both_8192x4096", "kind": "drop_both", "t": 8192, "d": 4096, "type": "bf16"},
        # the same of a small model at an odd width, forward
        {"name": "drop_999x515", "kind": "drop", "t": 999, "d": 515, "type": "f32"},
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _size(rng, lo, hi, step):
    """As `_between`; half of the time the nearest multiple of `step`, as users often choose."""
    v = _between(rng, lo, hi)
    return max(step, v // step * step) if rng.random() < 1 / 2 else v


def draw(rng):
    kind = rng.choice(("rotary", "rotary_both", "attn", "attn", "attn", "attn_both", "attn_both", "moe", "moe_both", "drop", "drop_both"))
    c = {"kind": kind, "type": rng.choice(("bf16", "bf16", "f16", "f32"))}
    if kind.startswith("rotary"):
        d = rng.choice((32, 64, 80, 96, 128, 128))
        hk = rng.choice((1, 2, 4, 8))
        c.update(t=_size(rng, 1, 8192, 64), hq=hk * rng.choice((1, 2, 3, 4)), hk=hk, d=d, r=rng.choice((d, d, d // 2)), half=rng.random() < 1 / 2,
                 norm=rng.random() < 2 / 3, far=rng.choice((0, 1000, 100000, 1000000)))
        c["t"] = min(c["t"], 8192 * 20 * 128 // ((c["hq"] + hk) * d))
    elif kind == "attn":
        hk = rng.choice((1, 2, 4, 8))
        c.update(n=_between(rng, 1, 64), hq=hk * rng.choice((1, 2, 3, 4, 8)), hk=hk, d=rng.choice((64, 64, 80, 96, 128, 128, 128)))
        form = rng.choice(("single", "single", "chunk", "prompt"))
        if form == "single":
            c["t"] = c["n"]
            c["tk"] = c["n"] * _between(rng, 1, 8192)
            c["tk"] = max(c["n"], min(c["tk"], 262144 * 8 * 128 // (hk * c["d"] * TYPES[c["type"]].itemsize // 2)))
        else:
            c["n"] = min(c["n"], 8)
            c["t"] = c["n"] * _size(rng, 8, 2048, 64)
            c["t"] = max(c["n"], min(c["t"], 16500 * 32 * 128 // (4 * c["hq"] * c["d"])))
            c["tk"] = c["t"] + (c["n"] * _between(rng, 16, 8192) if form == "chunk" else 0)
        c["w"] = rng.choice((-1, _between(rng, 64, 8192), _between(rng, 64, 2048)))
        c["sinks"] = rng.choice((0, 1, 4, 16)) if c["w"] > 0 else 0
    elif kind == "attn_both":
        hk = rng.choice((1, 2, 4))
        c.update(n=_between(rng, 1, 8), hq=hk * rng.choice((1, 2, 4)), hk=hk, d=rng.choice((64, 80, 128, 128)))
        c["t"] = c["n"] * _size(rng, 16, min(2048, 8192 // c["n"]), 64)
        c["t"] = max(c["n"], min(c["t"], 8192 * 16 * 128 // (c["hq"] * c["d"] * (4 if c["type"] == "f32" else 1))))
        c["tk"] = c["t"]
        c["w"] = rng.choice((-1, _between(rng, 64, 1024), _between(rng, 64, 1024)))
        c["sinks"] = rng.choice((0, 1, 4, 16)) if c["w"] > 0 else 0
    elif kind.startswith("moe"):
        c.update(k=rng.choice((1, 2, 2, 4, 8)), e=rng.choice((8, 16, 60, 128)), d=_size(rng, 64, 4096, 64))
        c["t"] = max(1, min(_size(rng, 1, 8192, 64), 8192 * 2 * 2048 // (c["k"] * c["d"])))
    else:
        c.update(t=_size(rng, 1, 8192, 64), d=_size(rng, 64, 4096, 64))
    return c


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------

def _cuts(total, n, turn):
    """Offsets of n uneven shares of `total`, the same for every seed."""
    share = [1.0 + 0.8 * math.cos(2.4 * i + turn) for i in range(n)]
    at, out = 0.0, [0]
    for v in share:
        at += v
        out.append(round(at / sum(share) * total))
    return out


def _lengths(case):
    """(offsets of the sequences' queries, of their keys): single tokens, or uneven shares."""
    n, t = case["n"], case["t"]
    q = list(range(n + 1)) if t == n else _cuts(t, n, 0.3)
    past = _cuts(case["tk"] - t, n, 1.7)
    return q, [a + b for a, b in zip(q, past)]


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    kind, dt = case["kind"], TYPES[case["type"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    if kind.startswith("rotary"):
        t, hq, hk, d = (case[a] for a in ("t", "hq", "hk", "d"))
        # queries and keys as they lie in one product's rows, with the values behind them
        s = {"x": normal(t, (hq + 2 * hk) * d)[:, :(hq + hk) * d]}
        far = case["far"]
        # a far batch's own places, or a sequence from its start
        s["pos"] = torch.randint(0, far, (t,), generator=g, device=DEV) if far else torch.arange(t, device=DEV)
        s["gq"], s["gk"] = (1.0 + 0.1 * torch.randn(d, generator=g, device=DEV) for _ in range(2)) if case["norm"] else (None, None)
        # radians a position, each pair its own
        s["freq"] = BASE ** (-2.0 * torch.arange(case["r"] // 2, dtype=torch.float64, device=DEV) / case["r"])
        if kind == "rotary_both":
            s["yb"] = normal(t, (hq + hk) * d)
        return s
    if kind.startswith("attn"):
        t, tk, hq, hk, d = (case[a] for a in ("t", "tk", "hq", "hk", "d"))
        qs, ks = _lengths(case)
        s = {"qstart": torch.tensor(qs, device=DEV), "kstart": torch.tensor(ks, device=DEV)}
        if t == tk:    # a training step's or a prompt's: one product's rows
            row = normal(t, (hq + 2 * hk) * d)
            s.update(q=row[:, :hq * d], k=row[:, hq * d:(hq + hk) * d], v=row[:, (hq + hk) * d:])
        else:          # keys and values of the past and the new tokens, side by side
            row = normal(tk, 2 * hk * d)
            s.update(q=normal(t, hq * d), k=row[:, :hk * d], v=row[:, hk * d:])
        if kind == "attn_both":
            s["yb"] = normal(t, hq * d)
        return s
    if kind.startswith("moe"):
        t, k, e, d = (case[a] for a in ("t", "k", "e", "d"))
        # a router's choice: the k largest of scores that favour some experts, one slot in fifty dropped
        score = torch.randn(t, e, generator=g, device=DEV) + 0.5 * torch.randn(e, generator=g, device=DEV)
        top, ids = torch.topk(score, k, dim=1)
        drop = torch.rand(t, k, generator=g, device=DEV) < 0.02
        s = {"ids": torch.where(drop, torch.zeros_like(ids), ids + 1), "p": torch.softmax(top, 1), "x": normal(t, d), "ys": normal(t * k, d)}
        if kind == "moe_both":
            s.update(yb=normal(t, d), xsb=normal(t * k, d))
        return s
    t, d = case["t"], case["d"]
    s = {"x": normal(t, d), "res": normal(t, d), "key": torch.randint(-2 ** 62, 2 ** 62, (2,), generator=g, device=DEV)}
    if kind == "drop_both":
        s["yb"] = normal(t, d)
    return s


def prepare(case, seed):
    """The inputs, and the arrays that a program keeps for the results."""
    s, kind, dt = _inputs(case, seed), case["kind"], TYPES[case["type"]]

    def new(*shape, dtype=dt):
        return torch.empty(*shape, dtype=dtype, device=DEV)

    if kind.startswith("rotary"):
        t, w, d = case["t"], (case["hq"] + case["hk"]) * case["d"], case["d"]
        s["y"] = new(t, w)
        if kind == "rotary_both":
            s["xb"] = new(t, w)
            s["gqb"], s["gkb"] = (new(d, dtype=torch.float32), new(d, dtype=torch.float32)) if case["norm"] else (None, None)
    elif kind.startswith("attn"):
        t, tk, hq, hk, d = (case[a] for a in ("t", "tk", "hq", "hk", "d"))
        s.update(y=new(t, hq * d), lse=new(t, hq, dtype=torch.float32), lengths=_lengths(case))
        if kind == "attn_both":
            row = new(t, (hq + 2 * hk) * d)
            s.update(qb=row[:, :hq * d], kb=row[:, hq * d:(hq + hk) * d], vb=row[:, (hq + hk) * d:])
    elif kind.startswith("moe"):
        t, k, e, d = (case[a] for a in ("t", "k", "e", "d"))
        s.update(order=new(t * k, dtype=torch.int64), place=new(t, k, dtype=torch.int64), start=new(e + 1, dtype=torch.int64), y=new(t, d))
        s["xs"] = torch.zeros(t * k, d, dtype=dt, device=DEV)     # rows behind the last expert's stay as they are
        if kind == "moe_both":
            s.update(xb=new(t, d), pb=new(t, k, dtype=torch.float32), ysb=torch.zeros(t * k, d, dtype=dt, device=DEV))
    else:
        s["y"] = new(case["t"], case["d"])
        if kind == "drop_both":
            s["xb"] = new(case["t"], case["d"])
    return case, s


# ------------------------------------------------------------------------------------------
# the plain forms, in 32 bits
# ------------------------------------------------------------------------------------------

def _turned(x, c, s, half):
    """The pairs of x (t, h, r) turned by the angles whose cosines and sines are c and s (t, 1, r / 2)."""
    if half:
        a, b = x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)


def _plain_rotary(case, s):
    t, hq, hk, d, r = (case[a] for a in ("t", "hq", "hk", "d", "r"))
    dt, out = TYPES[case["type"]], {}
    x = s["x"].float().reshape(t, hq + hk, d)
    angle = s["pos"].double()[:, None, None] * s["freq"]
    c, sn = torch.cos(angle).float(), torch.sin(angle).float()
    if case["norm"]:
        g = torch.cat([s["gq"].expand(hq, d), s["gk"].expand(hk, d)])
        rs = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        xh = x * rs
        h = xh * g
    else:
        h = x
    y = torch.cat([_turned(h[..., :r], c, sn, case["half"]), h[..., r:]], -1)
    out["y"] = y.reshape(t, -1).to(dt)
    if case["kind"] == "rotary_both":
        yb = s["yb"].float().reshape(t, hq + hk, d)
        hb = torch.cat([_turned(yb[..., :r], c, -sn, case["half"]), yb[..., r:]], -1)
        if case["norm"]:
            gb = (hb * xh).sum(0)
            out["gqb"], out["gkb"] = gb[:hq].sum(0), gb[hq:].sum(0)
            a = hb * g
            hb = rs * (a - xh * (a * xh).mean(-1, keepdim=True))
        out["xb"] = hb.reshape(t, -1).to(dt)
    return out


def _visible(p, nk, case):
    """Which of nk keys the queries at positions p see."""
    i = torch.arange(nk, device=DEV)
    seen = i <= p[..., None]
    if case["w"] >= 0:
        seen &= (p[..., None] - i < case["w"]) | (i < case["sinks"])
    return seen


def _plain_attn(case, s):
    hq, hk, d = (case[a] for a in ("hq", "hk", "d"))
    dt, both, scale, group = TYPES[case["type"]], case["kind"] == "attn_both", case["d"] ** -0.5, case["hq"] // case["hk"]
    qs, ks = s["lengths"]
    if case["t"] == case["n"]:    # single tokens: one padded batch
        n, nk = case["n"], s["kstart"][1:] - s["kstart"][:-1]
        longest = max(b - a for a, b in zip(ks, ks[1:]))
        at = (s["kstart"][:-1, None] + torch.arange(longest, device=DEV)).clamp_max(case["tk"] - 1)
        k = s["k"][at].float().reshape(n, longest, hk, d).transpose(1, 2).contiguous()
        v = s["v"][at].float().reshape(n, longest, hk, d).transpose(1, 2).contiguous()
        q = s["q"].float().reshape(n, hk, group, d)
        score = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
        score = score.masked_fill(~_visible(nk - 1, longest, case)[:, None, None, :], -torch.inf)
        top = score.amax(-1, keepdim=True)
        e = torch.exp(score - top)
        z = e.sum(-1, keepdim=True)
        y = torch.matmul(e / z, v)
        return {"y": y.reshape(n, hq * d).to(dt), "lse": (top + torch.log(z)).reshape(n, hq)}
    y, lse = torch.empty(case["t"], hq * d, dtype=dt, device=DEV), torch.empty(case["t"], hq, device=DEV)
    if both:
        qb, kb, vb = torch.empty_like(y), torch.empty(case["tk"], hk * d, dtype=dt, device=DEV), torch.empty(case["tk"], hk * d, dtype=dt, device=DEV)
    for a, b, ka, kz in zip(qs, qs[1:], ks, ks[1:]):
        nq, nk = b - a, kz - ka
        if nq == 0 and not both:
            continue
        k, v = (s[c][ka:kz].float().reshape(nk, hk, 1, d).permute(1, 2, 0, 3).contiguous() for c in "kv")       # (hk, 1, nk, d)
        kt = k.transpose(2, 3).contiguous()
        if both:
            k_sum, v_sum, vt = torch.zeros_like(k), torch.zeros_like(v), v.transpose(2, 3).contiguous()
        step = max(1, (1 << 28) // (hq * max(nk, 1)))       # rows whose scores take at most 1 GB
        for at in range(a, b, step):
            end = min(b, at + step)
            m = end - at
            q = s["q"][at:end].float().reshape(m, hk, group, d).permute(1, 2, 0, 3).contiguous()                  # (hk, group, m, d)
            score = torch.matmul(q, kt) * scale
            score = score.masked_fill(~_visible(nk - nq + torch.arange(at - a, end - a, device=DEV), nk, case), -torch.inf)
            top = score.amax(-1, keepdim=True)
            p = torch.exp(score - top)
            z = p.sum(-1, keepdim=True)
            p = p / z
            o = torch.matmul(p, v)
            y[at:end] = o.permute(2, 0, 1, 3).reshape(m, hq * d).to(dt)
            lse[at:end] = (top + torch.log(z)).permute(2, 0, 1, 3).reshape(m, hq)
            if both:
                ob = s["yb"][at:end].float().reshape(m, hk, group, d).permute(1, 2, 0, 3).contiguous()
                v_sum += torch.matmul(p.transpose(2, 3).contiguous(), ob).sum(1, keepdim=True)
                sb = p * (torch.matmul(ob, vt) - (o * ob).sum(-1, keepdim=True)) * scale
                qb[at:end] = torch.matmul(sb, k).permute(2, 0, 1, 3).reshape(m, hq * d).to(dt)
                k_sum += torch.matmul(sb.transpose(2, 3).contiguous(), q).sum(1, keepdim=True)
        if both:
            kb[ka:kz], vb[ka:kz] = (c.permute(2, 0, 1, 3).reshape(nk, hk * d).to(dt) for c in (k_sum, v_sum))
    return {"y": y, "lse": lse, "qb": qb, "kb": kb, "vb": vb} if both else {"y": y, "lse": lse}


def _plain_moe(case, s):
    t, k, e, d = (case[a] for a in ("t", "k", "e", "d"))
    dt, ids = TYPES[case["type"]], s["ids"].flatten()
    order = torch.sort(torch.where(ids > 0, ids, e + 1), stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(1, t * k + 1, device=DEV)
    place = torch.where(ids > 0, place, torch.zeros_like(place)).reshape(t, k)
    here = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), torch.cumsum(torch.bincount(ids, minlength=e + 1)[1:], 0)])
    full = (torch.arange(t * k, device=DEV) < here[-1])[:, None]
    out = {"place": place, "start": here, "xs": torch.where(full, s["x"][order // k], torch.zeros((), dtype=dt, device=DEV))}
    at, there = (place - 1).clamp_min(0), (place > 0)[..., None]

    def back(rows):     # (t, k, d), zeros for the dropped
        return torch.where(there, rows[at].float(), 0.0)

    y = back(s["ys"])
    out["y"] = (s["p"][..., None] * y).sum(1).to(dt)
    if case["kind"] == "moe_both":
        out["xb"] = back(s["xsb"]).sum(1).to(dt)
        yb = s["yb"].float()
        out["pb"] = (y * yb[:, None]).sum(-1)
        out["ysb"] = torch.where(full, (s["p"].flatten()[order][:, None] * yb[order // k]).to(dt), torch.zeros((), dtype=dt, device=DEV))
    return out


def _kept(key, t, d):
    """The mask of (t, d): Philox 4x32 with ten rounds, its key the first of `key`; eight values of a row share a
    block of 128 bits, whose counter is (their number in the row, the row, the second of `key`), and take 16
    bits each, which are kept from round(65536 p) on."""
    low = 0xFFFFFFFF
    k0, k1, c2, c3 = key[0] & low, (key[0] >> 32) & low, key[1] & low, (key[1] >> 32) & low
    m = -(-d // 8)
    c0, c1 = torch.arange(m, device=DEV).expand(t, m), torch.arange(t, device=DEV)[:, None].expand(t, m)
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57       # (the products' 64 bits, whatever their sign)
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    u = torch.stack([h for w in (c0, c1, c2, c3) for h in (w & 0xFFFF, w >> 16)], -1)
    return u.reshape(t, 8 * m)[:, :d] >= round(65536 * DROP)


def _plain_drop(case, s):
    dt, keep = TYPES[case["type"]], _kept(s["key"], case["t"], case["d"])
    scale = 65536.0 / (65536 - round(65536 * DROP))
    out = {"y": (s["res"].float() + torch.where(keep, s["x"].float() * scale, 0.0)).to(dt)}
    if case["kind"] == "drop_both":
        out["xb"] = torch.where(keep, s["yb"].float() * scale, 0.0).to(dt)
    return out


def _plain(case, s):
    kind = case["kind"].removesuffix("_both")
    return {"rotary": _plain_rotary, "attn": _plain_attn, "moe": _plain_moe, "drop": _plain_drop}[kind](case, s)


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
    both = kind.endswith("_both")
    if kind.startswith("rotary"):
        size = case["d"], case["hq"], case["hk"], case["r"], case["t"]
        form = dict(norm=case["norm"], eps=EPS, half=case["half"])
        hip.head_rotary(s["y"], s["x"], s["gq"], s["gk"], s["pos"], s["freq"], *size, **form)
        if not both:
            return {"y": s["y"]}
        hip.head_rotary_b(s["yb"], s["x"] if case["norm"] else None, s["xb"], s["gq"], s["gqb"], s["gk"], s["gkb"], s["pos"], s["freq"], *size,
                          add=False, **form)
        return {a: s[a] for a in (("y", "gqb", "gkb", "xb") if case["norm"] else ("y", "xb"))}
    if kind.startswith("attn"):
        size = case["d"], case["hq"], case["hk"], case["t"], case["tk"], case["n"]
        form = dict(window=None if case["w"] < 0 else case["w"], sinks=case["sinks"])
        hip.attention(s["y"], s["lse"], s["q"], s["k"], s["v"], s["qstart"], s["kstart"], case["d"] ** -0.5, *size, **form)
        if not both:
            return {a: s[a] for a in ("y", "lse")}
        hip.attention_b(s["yb"], s["y"], s["lse"], s["q"], s["qb"], s["k"], s["kb"], s["v"], s["vb"], s["qstart"], s["kstart"], case["d"] ** -0.5, *size,
                        add=False, **form)
        return {a: s[a] for a in ("y", "lse", "qb", "kb", "vb")}
    if kind.startswith("moe"):
        t, k, e, d = (case[a] for a in ("t", "k", "e", "d"))
        hip.expert_order(s["ids"], s["order"], s["place"], s["start"], k, e, t)
        hip.expert_take(s["xs"], s["x"], s["place"], d, k, t)
        hip.expert_join(s["y"], s["ys"], s["p"], s["place"], d, k, t)
        if both:
            hip.expert_join_b(s["yb"], s["ys"], s["ysb"], s["p"], s["pb"], s["place"], d, k, t, add=False)
            hip.expert_take_b(s["xsb"], s["xb"], s["place"], d, k, t, add=False)
        return {a: s[a] for a in ("place", "start", "xs", "y") + (("xb", "pb", "ysb") if both else ())}
    hip.dropout(s["y"], s["x"], s["res"], s["key"], DROP, case["d"], case["t"])
    if not both:
        return {"y": s["y"]}
    hip.dropout_b(s["yb"], s["xb"], s["key"], DROP, case["d"], case["t"], add=False)
    return {"y": s["y"], "xb": s["xb"]}


def run(state):
    return _own(*state) if own else _plain(*state)


# ------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------

def _pairs(case):
    """(visible pairs of a query and a key, keys that some query sees), over all sequences."""
    qs, ks = _lengths(case)
    pairs = keys = 0
    for a, b, ka, kz in zip(qs, qs[1:], ks, ks[1:]):
        nq, nk = b - a, kz - ka
        p = torch.arange(nk - nq, nk, dtype=torch.int64)
        if case["w"] < 0:
            pairs += int((p + 1).sum())
            keys += nk if nq else 0
            continue
        inside = torch.clamp(p + 1, max=case["w"])                                 # the window's
        sinks = torch.clamp(torch.clamp(p + 1 - case["w"], min=0), max=case["sinks"])    # sinks before it
        pairs += int((inside + sinks).sum())
        if nq:
            first = max(0, nk - nq + 1 - case["w"])
            keys += nk - first + min(first, case["sinks"])
    return pairs, keys


def work(case):
    kind, b = case["kind"], TYPES[case["type"]].itemsize
    both = kind.endswith("_both")
    if kind.startswith("rotary"):
        nd = case["t"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": float(nd * b * (2 + both * (2 + case["norm"])) + 8 * case["t"] * (1 + both)), "flops": float(nd * (9 + both * 14))}
    if kind.startswith("attn"):
        t, hq, hk, d = (case[a] for a in ("t", "hq", "hk", "d"))
        pairs, keys = _pairs(case)
        # forward: q, k, v in, y and lse out; reverse: yb, y, lse, q, k, v in, qb, kb, vb out
        size = 2 * t * hq * d * b + 2 * keys * hk * d * b + 4 * t * hq
        if both:
            size += 4 * t * hq * d * b + 4 * t * hq + 4 * keys * hk * d * b
        return {"bytes": float(size), "flops": float((4 + 10 * both) * pairs * hq * d)}
    if kind.startswith("moe"):
        t, k, d = (case[a] for a in ("t", "k", "d"))
        size = t * d * b * (1 + k + k + 1) + 8 * t * k * 2 + 4 * t * k + 8 * (case["e"] + 1)
        if both:    # yb, ys in, ysb out, xsb in, xb out
            size += t * d * b * (1 + k + k + k + 1) + 8 * t * k
        return {"bytes": float(size), "flops": float(2 * t * k * d * (1 + 2 * both))}
    nd = case["t"] * case["d"]
    return {"bytes": float(nd * b * (3 + 2 * both)), "flops": float(nd * (2 + both))}


# ------------------------------------------------------------------------------------------
# the same in 64 bits
# ------------------------------------------------------------------------------------------

def _exact_rotary(case, s):
    t, hq, hk, d, r = (case[a] for a in ("t", "hq", "hk", "d", "r"))
    leaves = {"x": s["x"].double().clone().requires_grad_()}
    if case["norm"]:
        leaves.update(gq=s["gq"].double().requires_grad_(), gk=s["gk"].double().requires_grad_())
    x, parts = leaves["x"], []
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["pos"].double()[:, None] * s["freq"])      # (t, r / 2)
    for h in range(hq + hk):
        v = x[:, h * d:(h + 1) * d]
        if case["norm"]:
            v = v / torch.sqrt((v ** 2).sum(1, keepdim=True) / d + EPS) * leaves["gq" if h < hq else "gk"]
        z = torch.complex(v[:, :r // 2], v[:, r // 2:r]) if case["half"] else torch.complex(v[:, 0:r:2], v[:, 1:r:2])
        z = z * turn
        parts += [z.real, z.imag] if case["half"] else [torch.view_as_real(z).reshape(t, r)]
        parts.append(v[:, r:])
    y = torch.cat(parts, 1)
    out = {"y": y.detach()}
    if case["kind"] == "rotary_both":
        (y * s["yb"].double()).sum().backward()
        if case["norm"]:
            out.update(gqb=leaves["gq"].grad, gkb=leaves["gk"].grad)
        out["xb"] = leaves["x"].grad
    return out


def _exact_attn(case, s):
    hq, hk, d = (case[a] for a in ("hq", "hk", "d"))
    both, group = case["kind"] == "attn_both", case["hq"] // case["hk"]
    if _pairs(case)[0] * hq * (1 + 3 * both) > 1 << 36:
        return None
    qs, ks = _lengths(case)
    zeros = lambda *n: torch.zeros(*n, dtype=torch.float64, device=DEV)   # noqa: E731
    out = {"y": zeros(case["t"], hq * d), "lse": zeros(case["t"], hq)}
    if both:
        out.update(qb=zeros(case["t"], hq * d), kb=zeros(case["tk"], hk * d), vb=zeros(case["tk"], hk * d))
    for a, b, ka, kz in zip(qs, qs[1:], ks, ks[1:]):
        nq, nk = b - a, kz - ka
        if nq == 0:
            continue
        far = torch.arange(nk - nq, nk, device=DEV)[:, None] - torch.arange(nk, device=DEV)     # how far back a key lies
        hidden = far < 0
        if case["w"] >= 0:
            hidden |= (far >= case["w"]) & (torch.arange(nk, device=DEV) >= case["sinks"])
        for kv in range(hk):
            cols = slice(kv * d, kv * d + d)
            k, v = (s[c][ka:kz, cols].double().clone().requires_grad_(both) for c in "kv")
            for h in range(kv * group, kv * group + group):
                mine = slice(h * d, h * d + d)
                q = s["q"][a:b, mine].double().clone().requires_grad_(both)
                score = (q @ k.t() / math.sqrt(d)).masked_fill(hidden, -math.inf)
                lse = torch.logsumexp(score, 1)
                y = torch.exp(score - lse[:, None]) @ v
                out["y"][a:b, mine], out["lse"][a:b, h] = y.detach(), lse.detach()
                if both:
                    (y * s["yb"][a:b, mine].double()).sum().backward()
                    out["qb"][a:b, mine] = q.grad
            if both:
                out["kb"][ka:kz, cols], out["vb"][ka:kz, cols] = k.grad, v.grad
    return out


def _exact_moe(case, s):
    t, k, e, d = (case[a] for a in ("t", "k", "e", "d"))
    flat = s["ids"].flatten().tolist()
    count = [0] * (e + 1)
    for i in flat:
        count[i] += 1
    start = [0]
    for c in count[1:]:
        start.append(start[-1] + c)
    at, place = list(start), []
    for i in flat:
        place.append(0 if i == 0 else at[i - 1] + 1)
        if i:
            at[i - 1] += 1
    place = torch.tensor(place, device=DEV)
    token, slot = torch.div(place.nonzero()[:, 0], k, rounding_mode="floor"), place[place > 0] - 1
    p, x, ys = s["p"].double().flatten()[place > 0], s["x"].double(), s["ys"].double()


    xs = torch.zeros(t * k, d, dtype=torch.float64, device=DEV).index_copy_(0, slot, x[token])
    y = torch.zeros(t, d, dtype=torch.float64, device=DEV).index_add_(0, token, p[:, None] * ys[slot])
    out = {"place": place.reshape(t, k), "start": torch.tensor(start, device=DEV), "xs": xs, "y": y}
    if case["kind"] == "moe_both":
        yb = s["yb"].double()
        out["xb"] = torch.zeros(t, d, dtype=torch.float64, device=DEV).index_add_(0, token, s["xsb"].double()[slot])
        pb = torch.zeros(t * k, dtype=torch.float64, device=DEV)
        pb[place > 0] = (ys[slot] * yb[token]).sum(1)
        out["pb"] = pb.reshape(t, k)
        out["ysb"] = torch.zeros(t * k, d, dtype=torch.float64, device=DEV).index_copy_(0, slot, p[:, None] * yb[token])
    return out


def _exact_drop(case, s):
    t, d = case["t"], case["d"]
    first, second = (int(v) & (1 << 64) - 1 for v in s["key"].tolist())
    mask, word = np.uint64(0xFFFFFFFF), np.uint64(32)
    m = (d + 7) // 8
    x = [np.tile(np.arange(m, dtype=np.uint64), t), np.repeat(np.arange(t, dtype=np.uint64), m), np.full(t * m, second & 0xFFFFFFFF, np.uint64),
         np.full(t * m, second >> 32, np.uint64)]
    key = [first & 0xFFFFFFFF, first >> 32]
    for _ in range(10):
        p, q = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(q >> word) ^ x[1] ^ np.uint64(key[0]), q & mask, (p >> word) ^ x[3] ^ np.uint64(key[1]), p & mask]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    bits = np.stack(x, 1).astype("<u4").view("<u2").reshape(t, 8 * m)[:, :d]
    least = round(65536 * DROP)
    scaled = torch.from_numpy(bits >= least).to(DEV).double() * 65536.0 / (65536.0 - least)
    out = {"y": s["res"].double() + s["x"].double() * scaled}
    if case["kind"] == "drop_both":
        out["xb"] = s["yb"].double() * scaled
    return out


def exact(case, seed):
    kind = case["kind"].removesuffix("_both")
    return {"rotary": _exact_rotary, "attn": _exact_attn, "moe": _exact_moe, "drop": _exact_drop}[kind](case, _inputs(case, seed))
