"""Shared by the attention tests: sequences, the formulas in 64 bits, and the bounds that the kernels' arithmetic gives.

Bounds are elementwise, to first order (lmhelp has the symbols).  A score s q . k is a product of d terms summed in fp32: off by
(d + 4) U s sum |q k|.  An exponential of a difference of scores is off by that, by the roundings of the
exponent's product and sum (4 U of their sizes) and by 4 U of its own, all relative; rounded to the type by half a step of it, and by
half a step of the type's least number, where it is below the type's normal range.  The hardware's (fp32) exponential is 0 where it
would be below 2^-126, so a weight w off by TINY = 2^-126 moves w x by TINY |x|, and a product of two factors that is itself below
2^-126 may be taken as 0: TINY (|x| + 1) a term."""
import torch

from lmhelp import LEAST, ROUND, U, gen, normal

TINY = 2.0 ** -126


class Case:
    """Sequences of (queries, keys) with `lead` columns of none before them and `tail` behind."""

    def __init__(self, seqs, hq, hk, d, window=None, sinks=0, dtype=torch.float32, lead=0, tail=0, seed=0, s=None):
        self.seqs, self.hq, self.hk, self.d, self.dtype = seqs, hq, hk, d, dtype
        self.window, self.sinks = window, sinks
        self.n, self.s = len(seqs), d ** -0.5 if s is None else s
        self.qs, self.ks = [lead], [lead]
        for nq, nk in seqs:
            self.qs.append(self.qs[-1] + nq)
            self.ks.append(self.ks[-1] + nk)
        self.t, self.tk = self.qs[-1] + tail, self.ks[-1] + tail
        g = gen(seed + 7 * self.t + d)
        self.q, self.yb = (normal(g, self.t, hq * d, dtype=dtype) for _ in range(2))
        self.k, self.v = (normal(g, self.tk, hk * d, dtype=dtype) for _ in range(2))

    def seen(self, i):
        """(queries, keys) truth values of sequence i."""
        nq, nk = self.seqs[i]
        p, key = torch.arange(nk - nq, nk)[:, None], torch.arange(nk)
        ok = key <= p
        if self.window is not None:
            ok &= (p - key < self.window) | (key < self.sinks)
        return ok

    def size(self):
        return self.d, self.hq, self.hk, self.t, self.tk, self.n

    def form(self):
        return dict(window=self.window, sinks=self.sinks)

    def starts(self):
        return torch.tensor(self.qs).cuda(), torch.tensor(self.ks).cuda()

    def forward(self, q=None, k=None, v=None, y=None, lse=None):
        import stade_hip
        y = torch.full((self.t, self.hq * self.d), float("nan"), dtype=self.dtype, device="cuda") if y is None else y
        lse = torch.full((self.t, self.hq), float("nan"), device="cuda") if lse is None else lse
        a = [b.cuda() if c is None else c for b, c in ((self.q, q), (self.k, k), (self.v, v))]
        stade_hip.attention(y, lse, *a, *self.starts(), self.s, *self.size(), **self.form())
        return y, lse

    def backward(self, y, lse, add=False, base=None, parts="qkv"):
        """(qb, kb, vb)"""
        import stade_hip
        like = dict(q=self.q, k=self.k, v=self.v)
        out = {a: (base[a].cuda() if add else torch.full_like(like[a], float("nan")).cuda()) if a in parts else None for a in "qkv"}
        stade_hip.attention_b(self.yb.cuda(), y, lse, self.q.cuda(), out["q"], self.k.cuda(), out["k"], self.v.cuda(), out["v"], *self.starts(), self.s,
                              *self.size(), add=add, **self.form())
        return out["q"], out["k"], out["v"]


def formula(c, grads=True):
    """The results in 64 bits and their bounds before rounding: dicts of y, lse, qb, kb, vb."""
    zeros = lambda n, w: torch.zeros(n, w, dtype=torch.float64)   # noqa: E731
    d, s, r, least = c.d, c.s, ROUND[c.dtype] if c.dtype != torch.float32 else 0.0, LEAST[c.dtype]
    tiny = TINY + (least if c.dtype != torch.float32 else 0)     # of a weight: the exponential's, and its rounding's
    out = {a: zeros(n, w) for a, n, w in (("y", c.t, c.hq * d), ("lse", c.t, c.hq), ("qb", c.t, c.hq * d), ("kb", c.tk, c.hk * d), ("vb", c.tk, c.hk * d))}
    out["lse"].fill_(-torch.inf)
    err = {a: torch.zeros_like(v) for a, v in out.items()}
    for i, (nq, nk) in enumerate(c.seqs):
        if nq == 0 or nk == 0:
            continue
        ok, rq, rk = c.seen(i), slice(c.qs[i], c.qs[i] + nq), slice(c.ks[i], c.ks[i] + nk)
        any_seen = ok.any(1)
        for h in range(c.hq):
            kv = h // (c.hq // c.hk)
            cq, ck = slice(h * d, h * d + d), slice(kv * d, kv * d + d)
            q, k, v, yb = (a.double() for a in (c.q[rq, cq], c.k[rk, ck], c.v[rk, ck], c.yb[rq, cq]))
            x = s * (q @ k.T)
            ex = (d + 4) * U * abs(s) * (q.abs() @ k.abs().T)
            xs = torch.where(ok, x, torch.full_like(x, -torch.inf))
            lse = torch.logsumexp(xs, 1)
            safe = torch.where(any_seen, lse, torch.zeros_like(lse))[:, None]
            p = torch.where(ok, torch.exp(x - safe), torch.zeros_like(x))
            top = torch.where(any_seen, xs.amax(1), torch.zeros_like(lse))[:, None]
            # of exp(x - m), m the running maximum
            ep = ex + 4 * U * (x.abs() + top.abs()) + 4 * U
            y = p @ v
            # the sums nest at most nk deep; what is scaled is rounded once a tile; weights below the least number of the type
            deep = (nk + 40) * U
            size = p @ v.abs() + y.abs()
            out["y"][rq, cq] = y
            ey = ((p * (ep + r)) @ v.abs()) + (p * (ep + r)).sum(1, keepdim=True) * y.abs() + deep * size
            ey = ey + tiny * (ok.double() @ (v.abs() + 1))
            err["y"][rq, cq] = ey
            out["lse"][rq, h] = lse
            el = (p * ep).sum(1) + deep + 4 * U * (safe[:, 0].abs() + top[:, 0].abs())
            err["lse"][rq, h] = torch.where(any_seen, el, torch.zeros_like(el))
            if not grads:
                continue
            # P again from lse, which was rounded
            e2 = ex + 4 * U * (x.abs() + safe.abs()) + el[:, None] + 6 * U
            delta = (yb * y).sum(1, keepdim=True)
            dp = yb @ v.T
            # y came rounded to the type
            edelta = (yb.abs() * (ey + ROUND[c.dtype] * y.abs() + least)).sum(1, keepdim=True) + (d + 4) * U * (yb * y).abs().sum(1, keepdim=True)
            edp = (d + 4) * U * (yb.abs() @ v.abs().T)
            w = p * (dp - delta)
            ew = p * (e2 * (dp - delta).abs() + edp + edelta) + (r + 4 * U) * w.abs()
            # (the weight times dp - delta, and their product rounded)
            ew = ew + TINY * (1 + (dp - delta).abs()) * ok + (least * ok if c.dtype != torch.float32 else 0)
            wide = (nq * c.hq // c.hk + 40) * U
            out["qb"][rq, cq] = s * (w @ k)
            err["qb"][rq, cq] = abs(s) * (ew @ k.abs() + deep * (w.abs() @ k.abs()) + TINY * nk)
            out["kb"][rk, ck] += s * (w.T @ q)
            err["kb"][rk, ck] += abs(s) * (ew.T @ q.abs() + wide * (w.abs().T @ q.abs()) + TINY * nq)
            out["vb"][rk, ck] += p.T @ yb
            evb = (p * (e2 + r)).T @ yb.abs() + wide * (p.T @ yb.abs())
            evb = evb + tiny * (ok.double().T @ (yb.abs() + 1))
            err["vb"][rk, ck] += evb
    return out, err
