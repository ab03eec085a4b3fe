"""Calls of attention and its surroundings captured in a HIP graph after one eager call of the function at its largest
size.  The scratch only grows within a process, so each case runs in one of its own."""
import subprocess
import sys

import pytest
import torch

import test_gpu_lm_capture as lm
from lmhelp import gen, normal

pytestmark = pytest.mark.gpu


def _attention(nq, nk, n, hq, hk, d, window, sinks, backward):
    import stade_hip as hip
    g = gen(nk)
    t, tk, dt = n * nq, n * nk, torch.bfloat16
    q, yb, k, v = (normal(g, r, h * d, dtype=dt).cuda() for r, h in ((t, hq), (t, hq), (tk, hk), (tk, hk)))
    qs, ks = (torch.arange(n + 1) * nq).cuda(), (torch.arange(n + 1) * nk).cuda()
    y, lse = torch.zeros_like(q), torch.zeros(t, hq, device="cuda")
    qb, kb, vb = (torch.zeros_like(a) for a in (q, k, v))
    form = dict(window=window, sinks=sinks)

    def call():
        hip.attention(y, lse, q, k, v, qs, ks, 0.1, d, hq, hk, t, tk, n, **form)
        if backward:
            hip.attention_b(yb, y, lse, q, qb, k, kb, v, vb, qs, ks, 0.1, d, hq, hk, t, tk, n, add=False, **form)
    return call, [y, lse] + ([qb, kb, vb] if backward else [])


def _order(t, k, e):
    import stade_hip as hip
    ids = torch.randint(0, e + 1, (t, k), generator=gen(t)).cuda()
    order, place, start = torch.zeros(t * k, dtype=torch.int64, device="cuda"), torch.zeros_like(ids), torch.zeros(e + 1, dtype=torch.int64, device="cuda")
    return lambda: hip.expert_order(ids, order, place, start, k, e, t), [order, place, start]


def _rotary_b(t, d, hq, hk):
    import stade_hip as hip
    g, width = gen(t), d * (hq + hk)
    x, yb = normal(g, t, width).cuda(), normal(g, t, width).cuda()
    w, pos, freq = torch.ones(d, device="cuda"), torch.arange(t).cuda(), torch.from_numpy(hip.rotary_freq(d)).cuda()
    xb, gqb, gkb = torch.zeros_like(x), torch.zeros(d, device="cuda"), torch.zeros(d, device="cuda")
    return lambda: hip.head_rotary_b(yb, x, xb, w, gqb, w, gkb, pos, freq, d, hq, hk, d, t, add=False), [xb, gqb, gkb]


CASES = {
    "attention": (_attention, (2000, 2000, 2, 8, 4, 128, None, 0, False), [(1, 2000, 2, 8, 4, 128, None, 0, False), (1, 1990, 1, 8, 1, 64, 1900, 4, False)]),
    "attention_b": (_attention, (1500, 1500, 2, 8, 4, 128, None, 0, True), [(700, 700, 2, 8, 4, 128, 100, 64, True), (300, 100, 1, 2, 1, 40, 90, 3, True)]),
    "expert_order": (_order, (3000, 2, 2000), [(2900, 2, 64), (10, 2, 8), (2999, 2, 2000)]),
    "head_rotary_b": (_rotary_b, (3000, 64, 4, 2), [(40, 256, 1, 1), (2999, 8, 2, 2)]),
}


def capture_after_largest(name):
    lm.CASES[name] = CASES[name]
    lm.capture_after_largest(name)


def first_calls():
    """Calls that use nothing of the library's are captured with no call before them."""
    import stade_hip as hip
    n, d = 40, 96
    g = gen(5)
    x, r = normal(g, n, d).cuda(), normal(g, n, d).cuda()
    y, z, xb = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    key, pos, freq = torch.tensor([1, 2]).cuda(), torch.arange(n).cuda(), torch.from_numpy(hip.rotary_freq(32)).cuda()

    def calls():
        hip.dropout(y, x, r, key, 0.25, d, n)
        hip.head_rotary(z, x, None, None, pos, freq, 32, 2, 1, 32, n)
        hip.head_rotary_b(r, x, xb, None, None, None, None, pos, freq, 32, 2, 1, 32, n, add=False)
        hip.dropout_b(xb, xb, key, 0.25, d, n, add=False)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    calls()
    torch.cuda.synchronize()
    outs = [y, z, xb]
    eager = [v.clone() for v in outs]
    for rep in range(3):
        for v in outs:
            v.fill_(3)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(v, w) for v, w in zip(outs, eager)), f"replay {rep}"
        _ = torch.randn(1000, device="cuda").sum().item()
    print("captured", flush=True)


def _in_a_process(call):
    from helpers import ROOT
    code = (f"import sys; sys.path[:0] = [{str(ROOT / 'tests')!r}, {str(ROOT / 'stade.jl_amd')!r}]; "
            f"import test_gpu_attention_capture as m; m.{call}")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100, cwd=str(ROOT))
    assert r.returncode == 0 and "captured" in r.stdout.split(), r.stdout[-2000:] + r.stderr[-2000:]


def test_first_calls_that_need_no_workspace():
    print("capture without an eager call: dropout, head_rotary", flush=True)
    _in_a_process("first_calls()")


@pytest.mark.parametrize("name", CASES)
def test_smaller_calls_are_captured_after_the_largest(name):
    print(f"capture after the largest call: {name}", flush=True)
    _in_a_process(f"capture_after_largest({name!r})")
