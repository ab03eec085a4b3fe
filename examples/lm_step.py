"""A small language model trained with the operators of stade_hip, as a program uses them together:

    tokens -> rows (embed) -> layer norm -> products by expert -> least squares to a target

Every step runs the primal functions, then the adjoints in reverse order, then plain gradient descent.  What
the reverse sweep needs of the layer norm's input and of the experts' input is held in 8 bits.  Each token
is sent to one expert by a fixed random table (a router's choice).

    python examples/lm_step.py            # needs the built library and a GPU
"""
import sys
from pathlib import Path

import torch

PKG = Path(__file__).resolve().parent.parent / "stade.jl_amd"
if str(PKG) not in sys.path:
    sys.path.insert(0, str(PKG))

import stade_hip as hip  # noqa: E402

SCALE = 4.0   # of the embedding rows


class Model:
    """Weights, and the arrays that one step keeps: activations, their tapes and the shadows."""

    def __init__(self, t=512, d=256, o=128, v=1000, e=8, dtype=torch.bfloat16, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.t, self.d, self.o, self.v, self.e = t, d, o, v, e
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g)   # noqa: E731
        # master weights in Float32, working copies in `dtype`
        self.table, self.w = 0.25 * rand(v, d), rand(e, d, o) * d ** -0.5
        self.gain, self.bias = torch.ones(d, device="cuda"), torch.zeros(d, device="cuda")
        self.expert_of = torch.randint(1, e + 1, (v,), device="cuda", generator=g)
        new = lambda *s, dt=dtype: torch.empty(*s, dtype=dt, device="cuda")   # noqa: E731
        f32, i64 = torch.float32, torch.int64
        self.x, self.n, self.ns, self.y = new(t, d), new(t, d), new(t, d), new(t, o)
        self.mu, self.rs = new(t, dt=f32), new(t, dt=f32)
        self.order, self.start = new(t, dt=i64), new(e + 1, dt=i64)
        lq, ls = hip.tape8_lengths(d, t)
        self.tape_x, self.tape_ns = ((new(lq, dt=torch.int8), new(ls, dt=torch.uint8)) for _ in range(2))
        self.yb, self.nsb, self.nb, self.xb = new(t, o), new(t, d), new(t, d), new(t, d)
        self.tableb, self.wb, self.gainb, self.biasb = (torch.zeros_like(p) for p in (self.table, self.w, self.gain, self.bias))

    def forward(self, tok):
        t, d, o, v, e = self.t, self.d, self.o, self.v, self.e
        hip.embed(self.x, self.table, tok, SCALE, d, v, t)
        hip.layernorm(self.n, self.x, self.gain, self.bias, self.mu, self.rs, d, t, tape=self.tape_x)
        # rows in the order of their experts
        hip.token_order(self.expert_of[tok - 1], self.order, self.start, e, t)
        hip.embed(self.ns, self.n, self.order, 1.0, d, t, t)
        hip.tape8_store(self.ns, *self.tape_ns, d, t)
        self.wh = self.w.to(self.ns.dtype)
        hip.expert_mul(self.y, self.ns, self.wh, self.start, d, o, t, e)

    def backward(self, tok):
        """Shadows from yb: set, not accumulated (add=False), as each is the step's first and only use."""
        t, d, o, v, e = self.t, self.d, self.o, self.v, self.e
        hip.expert_mul_b(self.yb, None, self.nsb, self.wh, self.wb, self.start, d, o, t, e, add=False, tape=self.tape_ns)
        hip.embed_b(self.nsb, self.nb, self.order, 1.0, d, t, t, add=False)
        hip.layernorm_b(self.nb, None, self.xb, self.gain, self.gainb, self.biasb, self.mu, self.rs, d, t, add=False, tape=self.tape_x)
        hip.embed_b(self.xb, self.tableb, tok, SCALE, d, v, t, add=False)

    def step(self, tok, target, rate):
        """One training step; returns the loss before it (mean squared error over rows and columns)."""
        self.forward(tok)
        diff = self.y.float() - target[self.order - 1]
        self.yb.copy_(diff * (2.0 / diff.numel()))
        self.backward(tok)
        for p, b in ((self.table, self.tableb), (self.w, self.wb), (self.gain, self.gainb), (self.bias, self.biasb)):
            p.sub_(b, alpha=rate)
        return diff.square().mean()


def main(steps=60, rate=20.0):
    m = Model()
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    tok = torch.randint(1, m.v + 1, (m.t,), device="cuda", generator=g)
    target = torch.randn(m.v, m.o, device="cuda", generator=g)[tok - 1]   # (each token has a target of its own)
    losses = [m.step(tok, target, rate) for _ in range(steps)]
    losses = [float(v) for v in losses]
    for k in range(0, steps, max(1, steps // 6)):
        print(f"step {k:3d}  loss {losses[k]:.4f}", flush=True)
    print(f"step {steps - 1:3d}  loss {losses[-1]:.4f}", flush=True)
    return losses


if __name__ == "__main__":
    main()
