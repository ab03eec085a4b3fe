"""The operators of a block together, as the example runs them: a step's gradients against torch's own in 64 bits, on another
stream, and captured in a graph."""
import importlib.util

import pytest
import torch

from helpers import ROOT

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("block_step", ROOT / "examples" / "block_step.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _tokens(m, seed=3):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randint(1, m.v + 1, (m.t,), generator=g).cuda()


def _norm(x, g, b):
    mu = x.mean(1, keepdim=True)
    return (x - mu) / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + 1e-5) * g + b


def _plain(m, tok, lengths, keep):
    """(y, weights with gradients to come) in 64 bits, with the example's choice of experts and its mask."""
    w = {k: v.double().cpu().requires_grad_() for k, v in m.w.items()}
    t, d, hq, hk, a, c = m.t, m.d, m.hq, m.hk, m.a, m.c
    x = 4.0 * w["table"][tok.cpu() - 1]
    qkv = _norm(x, w["g1"], w["b1"]) @ w["in"][0]
    qk = qkv[:, :c].reshape(t, hq + hk, d)
    gain = torch.cat([w["gq"].expand(hq, d), w["gk"].expand(hk, d)])
    qk = qk / torch.sqrt((qk ** 2).mean(2, keepdim=True) + 1e-6) * gain
    angle = (m.pos.cpu()[:, None] * m.freq.cpu())[:, None]
    lo, hi = qk[..., :d // 2], qk[..., d // 2:]
    qk = torch.cat([lo * angle.cos() - hi * angle.sin(), lo * angle.sin() + hi * angle.cos()], 2)
    parts, at = [], 0
    for n in lengths:
        q, k, v = qk[at:at + n, :hq], qk[at:at + n, hq:], qkv[at:at + n, c:].reshape(n, hk, d)
        i, j = torch.arange(n)[:, None], torch.arange(n)
        seen = (j <= i) & ((i - j < m.window) | (j < m.sinks))
        k, v = (u.repeat_interleave(hq // hk, 1) for u in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * d ** -0.5
        parts.append(torch.einsum("hij,jhd->ihd", s.masked_fill(~seen, -torch.inf).softmax(2), v).reshape(n, a))
        at += n
    o2 = torch.cat(parts) @ w["out"][0]
    x2 = x + o2 * keep
    n2 = _norm(x2, w["g2"], w["b2"])
    ids = m.ids.cpu() - 1
    p = (n2 @ w["route"]).gather(1, ids).softmax(1)
    y = x2 + sum(p[:, k:k + 1] * torch.einsum("ti,tio->to", n2, w["expert"][ids[:, k]]) for k in range(m.k))
    return y, w


def test_step_against_torch():
    import stade_hip as hip
    lengths = (50, 1, 33, 90)
    m = _example().Block(lengths, dim=96, heads=6, kv_heads=2, head=32, window=20, sinks=2, experts=5, v=120, drop=0.2, dtype=torch.float32, seed=2)
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    for k in ("g1", "b1", "g2", "b2", "gq", "gk"):
        m.w[k] += 0.1 * torch.randn(m.w[k].shape, device="cuda", generator=g)
    tok = _tokens(m)
    print("block step", flush=True)
    m.forward(tok)
    m.yb.copy_(torch.randn(m.t, m.dim, device="cuda", generator=g))
    m.backward(tok)
    keep = torch.empty(m.t, m.dim, device="cuda")
    hip.dropout(keep, torch.ones_like(keep), None, m.key, m.drop, m.dim, m.t)
    assert 0.7 < (keep > 0).float().mean() < 0.9
    y, w = _plain(m, tok, lengths, keep.double().cpu())
    (y * m.yb.double().cpu()).sum().backward()
    # Twenty-odd operators one after the other in fp32: each sum of up to some 200 terms is off by at most 200 U = 1.2e-5 of the
    # sum of their sizes, some ten times the norm of what terms of both signs leave at the worst: 20 * 1.2e-5 in all, were all errors
    # of one sign at once.
    for name, got, want in [("y", m.y, y.detach())] + [(k, m.wb[k], w[k].grad) for k in m.w]:
        off = (got.double().cpu() - want).norm() / want.norm()
        assert off <= 2.4e-4, f"{name}: {off}"


def _fixed(m, tok):
    """The step with the router's choice as it is."""
    m.rows(tok)
    m.experts()
    for k in ("g1", "b1", "g2", "b2"):
        m.wb[k].zero_()
    m.experts_b()
    m.rows_b(tok)


def _results(m):
    return {"y": m.y, "pb": m.pb, "place": m.place, "xb": m.xb, "lse": m.lse, **{f"wb {k}": v for k, v in m.wb.items() if k != "route"}}


def _block(seed, **kw):
    m = _example().Block(seed=seed, **kw)
    tok = _tokens(m, seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    m.rows(tok)
    m.route()
    m.yb.copy_(torch.randn(m.t, m.dim, device="cuda", generator=g))
    return m, tok


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_graph_replays_match_eager(dt):
    m, tok = _block(5, dtype=dt)
    _fixed(m, tok)
    torch.cuda.synchronize()
    eager = {k: v.clone() for k, v in _results(m).items()}
    print("block step in a graph", flush=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _fixed(m, tok)
    for rep in range(3):
        for v in _results(m).values():
            v.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k, v in _results(m).items():
            assert torch.equal(v, eager[k]), f"replay {rep}: {k}"
        other, tok2 = _block(6, dtype=dt)      # (shares the library's workspace)
        _fixed(other, tok2)


def test_two_graphs_share_the_workspace():
    """Two captured steps of different sizes, replayed in turn, leave each other's results alone."""
    made = []
    for seed, lengths in ((7, (300, 20)), (8, (5, 700, 1, 64))):
        m, tok = _block(seed, lengths=lengths)
        _fixed(m, tok)
        made.append((m, tok))
    graphs = []
    for m, tok in made:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _fixed(m, tok)
        graphs.append(graph)
    want = []
    for m, tok in made:
        _fixed(m, tok)
        torch.cuda.synchronize()
        want.append({k: v.clone() for k, v in _results(m).items()})
    print("two graphs in turn", flush=True)
    for rep in range(3):
        for m, _ in made:
            for v in _results(m).values():
                v.zero_()
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (m, _), w in zip(made, want):
            assert all(torch.equal(v, w[k]) for k, v in _results(m).items()), rep


def test_other_stream():
    a, tok = _block(1)
    _fixed(a, tok)
    torch.cuda.synchronize()
    want = {k: v.clone() for k, v in _results(a).items()}
    b, _ = _block(1)
    c, tok2 = _block(2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    print("block step on a side stream", flush=True)
    with torch.cuda.stream(side):
        _fixed(b, tok)
    _fixed(c, tok2)        # shares the library's workspace with the calls on the side stream
    torch.cuda.synchronize()
    other = {k: v.clone() for k, v in _results(c).items()}
    for k, v in _results(b).items():
        assert torch.equal(v, want[k]), k
    _fixed(c, tok2)
    for k, v in _results(c).items():
        assert torch.equal(v, other[k]), k


def test_example_runs():
    print("block example", flush=True)
    losses = _example().main(steps=3)
    assert len(losses) == 3 and all(v == v and v < float("inf") for v in losses)
