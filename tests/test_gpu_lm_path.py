"""The language-model operators together: a small model's step through all of them against torch's
own gradients in 64 bits; on another stream than the tensors' own; and captured in a graph."""
import pytest
import torch

from lmhelp import gen, new_tape, normal

pytestmark = pytest.mark.gpu


class Step:
    """tokens -> rows -> layer norm -> products by expert, and the reverse sweep of
    loss = <y, c>, the layer norm's input held in 8 bits."""

    def __init__(self, t=200, d=96, o=64, v=150, e=5, dtype=torch.float32, seed=0):
        g = gen(seed)
        self.size = t, d, o, v, e
        self.tok = torch.randint(0, v + 1, (t,), generator=g).cuda()
        self.to = torch.randint(1, e + 1, (t,), generator=g).cuda()
        self.table, self.w = normal(g, v, d, dtype=dtype).cuda(), normal(g, e, d, o, dtype=dtype, scale=d ** -0.5).cuda()
        self.g, self.b = (1 + 0.1 * torch.randn(d, generator=g)).cuda(), (0.1 * torch.randn(d, generator=g)).cuda()
        self.c = normal(g, t, o, dtype=dtype).cuda()
        new = lambda *s, dt=dtype: torch.zeros(*s, dtype=dt, device="cuda")   # noqa: E731
        self.x, self.n, self.ns, self.y = new(t, d), new(t, d), new(t, d), new(t, o)
        self.mu, self.rs = new(t, dt=torch.float32), new(t, dt=torch.float32)
        self.order, self.start = new(t, dt=torch.int64), new(e + 1, dt=torch.int64)
        self.tape_x, self.tape_n = new_tape(d, t), new_tape(d, t)
        self.nsb, self.nb, self.xb = new(t, d), new(t, d), new(t, d)
        self.wb, self.gb, self.bb, self.tableb = new(e, d, o, dt=torch.float32), new(d, dt=torch.float32), new(d, dt=torch.float32), new(v, d, dt=torch.float32)

    def run(self):
        import stade_hip as hip
        t, d, o, v, e = self.size
        hip.embed(self.x, self.table, self.tok, 4.0, d, v, t)
        hip.layernorm(self.n, self.x, self.g, self.b, self.mu, self.rs, d, t, tape=self.tape_x)
        hip.token_order(self.to, self.order, self.start, e, t)
        hip.embed(self.ns, self.n, self.order, 1.0, d, t, t)
        hip.tape8_store(self.ns, *self.tape_n, d, t)
        hip.expert_mul(self.y, self.ns, self.w, self.start, d, o, t, e)
        hip.expert_mul_b(self.c, None, self.nsb, self.w, self.wb, self.start, d, o, t, e, add=False, tape=self.tape_n)
        hip.embed_b(self.nsb, self.nb, self.order, 1.0, d, t, t, add=False)
        hip.layernorm_b(self.nb, None, self.xb, self.g, self.gb, self.bb, self.mu, self.rs, d, t, add=False, tape=self.tape_x)
        hip.embed_b(self.xb, self.tableb, self.tok, 4.0, d, v, t, add=False)

    def results(self):
        return {k: getattr(self, k) for k in ("y", "xb", "wb", "gb", "bb", "tableb", "order", "start")}


def test_step_against_torch():
    s = Step()
    t, d, o, v, e = s.size
    print("language-model step", flush=True)
    s.run()
    table, w, g, b = (x.double().cpu().requires_grad_() for x in (s.table, s.w, s.g, s.b))
    tok, to, c = s.tok.cpu(), s.to.cpu(), s.c.double().cpu()
    x = 4.0 * torch.cat([torch.zeros(1, d, dtype=torch.float64), table])[tok]
    mu = x.mean(1, keepdim=True)
    n = (x - mu) / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + 1e-5) * g + b
    order = torch.sort(to, stable=True).indices
    y = torch.stack([n[i] @ w[to[i] - 1] for i in order.tolist()])
    (y * c).sum().backward()
    near = lambda a, want, most: (a.double().cpu() - want).norm() <= most * want.norm()   # noqa: E731
    assert torch.equal(s.order.cpu(), order + 1)
    # fp32 through three operators; the tapes' values are off by at most half a unit in 127 of the
    # largest of 32 (about 2.1 of their root mean square): 2.1 / 127 / sqrt(12) to 2 / 127 / sqrt(12) ... 0.5 %
    # of a value's size, twice that where the scale is just past its step, and no more in the gradients
    assert near(s.y, y.detach(), 1e-5)
    for got, want in ((s.wb, w.grad), (s.gb, g.grad), (s.tableb, table.grad)):
        assert near(got, want, 0.02)
    assert near(s.bb, b.grad, 1e-5)


def test_other_stream():
    """Calls on a side stream, with the tensors made on the default one: the results of the
    default stream, also for calls that follow on it at once."""
    a, b = Step(dtype=torch.bfloat16, seed=1), Step(dtype=torch.bfloat16, seed=1)
    a.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    print("language-model step on a side stream", flush=True)
    with torch.cuda.stream(side):
        b.run()
    other = Step(dtype=torch.bfloat16, seed=2)
    other.run()        # shares the library's workspace with the calls on the side stream
    torch.cuda.synchronize()
    for k, want in a.results().items():
        assert torch.equal(getattr(b, k), want), k
    again = Step(dtype=torch.bfloat16, seed=2)
    again.run()
    for k, want in again.results().items():
        assert torch.equal(getattr(other, k), want), k


def test_graph_replays_match_eager():
    s = Step(dtype=torch.bfloat16, seed=3)
    s.run()
    torch.cuda.synchronize()
    eager = {k: v.clone() for k, v in s.results().items()}
    print("language-model step in a graph", flush=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.run()
    for rep in range(3):
        for v in s.results().values():
            v.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for k, v in s.results().items():
            assert torch.equal(v, eager[k]), f"replay {rep}: {k}"
        _ = torch.randn(1000, device="cuda").sum().item()


def test_example_learns():
    """The example's model fits its tokens' targets: the loss falls at first and ends below a half of
    its start (no bound on how far: plain gradient descent)."""
    import importlib.util
    from helpers import ROOT
    spec = importlib.util.spec_from_file_location("lm_step", ROOT / "examples" / "lm_step.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    print("language-model example", flush=True)
    losses = mod.main(steps=40)
    assert losses[1] < losses[0] and losses[-1] < 0.5 * losses[0], losses
