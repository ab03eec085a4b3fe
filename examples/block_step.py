"""A block of a language model with the operators of stade_hip, as a program uses them together:

    tokens -> rows (embed) -> layer norm -> queries, keys and values -> their positions (head_rotary) -> attention over
    sequences of different lengths -> product -> dropout and residual -> layer norm -> each row to two experts and back

Every step runs the primal functions, then the adjoints in reverse order, then plain gradient descent.  Dense products
are products by expert with one expert.  The router's small product, its softmax and its choice are torch's.

    python examples/block_step.py         # needs the built library and a GPU
"""
import sys
from pathlib import Path

import torch

PKG = Path(__file__).resolve().parent.parent / "stade.jl_amd"
if str(PKG) not in sys.path:
    sys.path.insert(0, str(PKG))

import stade_hip as hip  # noqa: E402

SCALE = 4.0   # of the embedding rows


class Block:
    """Weights (Float32, with working copies in `dtype`), and the arrays that one step keeps."""

    def __init__(self, lengths=(100, 37, 250), dim=256, heads=4, kv_heads=2, head=64, window=64, sinks=2, experts=8, slots=2, v=500, drop=0.1,
                 dtype=torch.bfloat16, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.n, self.t, self.dim, self.hq, self.hk, self.d = len(lengths), sum(lengths), dim, heads, kv_heads, head
        self.window, self.sinks, self.e, self.k, self.v, self.drop = window, sinks, experts, slots, v, drop
        t, a, c = self.t, heads * head, (heads + kv_heads) * head
        b = c + kv_heads * head
        self.a, self.b, self.c = a, b, c
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g)   # noqa: E731
        one = lambda n: torch.ones(n, device="cuda")   # noqa: E731
        self.w = {"table": 0.25 * rand(v, dim), "in": rand(1, dim, b) * dim ** -0.5, "out": rand(1, a, dim) * a ** -0.5,
                  "route": rand(dim, experts) * dim ** -0.5, "expert": rand(experts, dim, dim) * dim ** -0.5,
                  "g1": one(dim), "b1": 0 * one(dim), "g2": one(dim), "b2": 0 * one(dim), "gq": one(head), "gk": one(head)}
        self.wb = {k: torch.zeros_like(w) for k, w in self.w.items()}
        new = lambda *s, dt=dtype: torch.zeros(*s, dtype=dt, device="cuda")   # noqa: E731
        f32, i64 = torch.float32, torch.int64
        start = torch.tensor([0, *lengths]).cumsum(0)
        self.start, self.whole = start.cuda(), torch.tensor([0, t]).cuda()
        self.pos = torch.cat([torch.arange(n) for n in lengths]).cuda()
        self.freq = torch.from_numpy(hip.rotary_freq(head)).cuda()
        self.key = torch.tensor([seed, 0], device="cuda")   # (seed, step)
        self.x, self.n1, self.o2, self.x2, self.n2, self.y = (new(t, dim) for _ in range(6))
        self.qkv, self.qk, self.o, self.lse = new(t, b), new(t, c), new(t, a), new(t, heads, dt=f32)
        self.stats = [new(t, dt=f32) for _ in range(4)]
        self.ids, self.p = new(t, slots, dt=i64), new(t, slots, dt=f32)
        self.order, self.place, self.first = new(t * slots, dt=i64), new(t, slots, dt=i64), new(experts + 1, dt=i64)
        self.xs, self.ys, self.xsb, self.ysb = (new(t * slots, dim) for _ in range(4))
        self.pb, self.scoreb = new(t, slots, dt=f32), new(t, experts, dt=f32)
        self.yb, self.n2b, self.x2b, self.o2b, self.n1b, self.xb = (new(t, dim) for _ in range(6))
        self.qkvb, self.qkb, self.ob = new(t, b), new(t, c), new(t, a)

    def rows(self, tok):
        """Everything before the router."""
        t, dim, w, a, c = self.t, self.dim, self.w, self.a, self.c
        self.wh = {k: w[k].to(self.x.dtype) for k in ("in", "out", "expert")}
        hip.embed(self.x, w["table"], tok, SCALE, dim, self.v, t)
        hip.layernorm(self.n1, self.x, w["g1"], w["b1"], *self.stats[:2], dim, t)
        hip.expert_mul(self.qkv, self.n1, self.wh["in"], self.whole, dim, self.b, t, 1)
        hip.head_rotary(self.qk, self.qkv[:, :c], w["gq"], w["gk"], self.pos, self.freq, self.d, self.hq, self.hk, self.d, t)
        hip.attention(self.o, self.lse, self.qk[:, :a], self.qk[:, a:], self.qkv[:, c:], self.start, self.start, self.d ** -0.5, self.d, self.hq, self.hk,
                      t, t, self.n, window=self.window, sinks=self.sinks)
        hip.expert_mul(self.o2, self.o, self.wh["out"], self.whole, a, dim, t, 1)
        hip.dropout(self.x2, self.o2, self.x, self.key, self.drop, dim, t)
        hip.layernorm(self.n2, self.x2, w["g2"], w["b2"], *self.stats[2:], dim, t)

    def route(self):
        """The choice of experts, and their weights."""
        top, at = (self.n2.float() @ self.w["route"]).topk(self.k, 1)
        self.ids.copy_(at + 1)
        self.p.copy_(top.softmax(1))

    def experts(self):
        t, dim, e, k = self.t, self.dim, self.e, self.k
        hip.expert_order(self.ids, self.order, self.place, self.first, k, e, t)
        hip.expert_take(self.xs, self.n2, self.place, dim, k, t)
        hip.expert_mul(self.ys, self.xs, self.wh["expert"], self.first, dim, dim, k * t, e)
        self.y.copy_(self.x2)
        hip.expert_join(self.y, self.ys, self.p, self.place, dim, k, t, add=True)

    def experts_b(self):
        """Shadows from yb: set where it is their first use."""
        t, dim, e, k = self.t, self.dim, self.e, self.k
        hip.expert_join_b(self.yb, self.ys, self.ysb, self.p, self.pb, self.place, dim, k, t, add=False)
        hip.expert_mul_b(self.ysb, self.xs, self.xsb, self.wh["expert"], self.wb["expert"], self.first, dim, dim, k * t, e, add=False)
        hip.expert_take_b(self.xsb, self.n2b, self.place, dim, k, t, add=False)

    def route_b(self):
        topb = self.p * (self.pb - (self.p * self.pb).sum(1, keepdim=True))
        self.scoreb.zero_().scatter_(1, self.ids - 1, topb)
        self.wb["route"].copy_(self.n2.float().T @ self.scoreb)
        self.n2b += (self.scoreb @ self.w["route"].T).to(self.n2b.dtype)

    def rows_b(self, tok):
        t, dim, w, wb, a, c = self.t, self.dim, self.w, self.wb, self.a, self.c
        self.x2b.copy_(self.yb)
        hip.layernorm_b(self.n2b, self.x2, self.x2b, w["g2"], wb["g2"], wb["b2"], *self.stats[2:], dim, t)
        # the residual's shadow is x2b itself
        hip.dropout_b(self.x2b, self.o2b, self.key, self.drop, dim, t, add=False)
        hip.expert_mul_b(self.o2b, self.o, self.ob, self.wh["out"], wb["out"], self.whole, a, dim, t, 1, add=False)
        hip.attention_b(self.ob, self.o, self.lse, self.qk[:, :a], self.qkb[:, :a], self.qk[:, a:], self.qkb[:, a:], self.qkv[:, c:], self.qkvb[:, c:],
                        self.start, self.start, self.d ** -0.5, self.d, self.hq, self.hk, t, t, self.n, window=self.window, sinks=self.sinks, add=False)
        hip.head_rotary_b(self.qkb, self.qkv[:, :c], self.qkvb[:, :c], w["gq"], wb["gq"], w["gk"], wb["gk"], self.pos, self.freq, self.d, self.hq, self.hk,
                          self.d, t, add=False)
        hip.expert_mul_b(self.qkvb, self.n1, self.n1b, self.wh["in"], wb["in"], self.whole, dim, self.b, t, 1, add=False)
        self.xb.copy_(self.x2b)
        hip.layernorm_b(self.n1b, self.x, self.xb, w["g1"], wb["g1"], wb["b1"], *self.stats[:2], dim, t)
        hip.embed_b(self.xb, wb["table"], tok, SCALE, dim, self.v, t, add=False)

    def forward(self, tok):
        self.rows(tok)
        self.route()
        self.experts()

    def backward(self, tok):
        for k in ("g1", "b1", "g2", "b2"):
            self.wb[k].zero_()
        self.experts_b()
        self.route_b()
        self.rows_b(tok)

    def step(self, tok, target, rate):
        """One training step; returns the loss before it (mean squared error over rows and columns)."""
        self.forward(tok)
        diff = self.y.float() - target
        self.yb.copy_(diff * (2.0 / diff.numel()))
        self.backward(tok)
        for k, w in self.w.items():
            w.sub_(self.wb[k], alpha=rate)
        self.key[1] += 1     # (another mask the next time)
        return diff.square().mean()


def main(steps=60, rate=1.0):
    m = Block()
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    tok = torch.randint(1, m.v + 1, (m.t,), device="cuda", generator=g)
    target = torch.randn(m.v, m.dim, device="cuda", generator=g)[tok - 1]   # (each token has a target of its own)
    losses = [m.step(tok, target, rate) for _ in range(steps)]
    losses = [float(v) for v in losses]
    for k in range(0, steps, max(1, steps // 6)):
        print(f"step {k:3d}  loss {losses[k]:.4f}", flush=True)
    print(f"step {steps - 1:3d}  loss {losses[-1]:.4f}", flush=True)
    return losses


if __name__ == "__main__":
    main()
