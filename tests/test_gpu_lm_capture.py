"""Calls captured in a HIP graph after one eager call of the function at its largest size: smaller ones
may take scratch where the largest takes none, or more of it, and are captured all the same.

The scratch only grows within a process, so each case runs in one of its own."""
import subprocess
import sys

import pytest
import torch

from lmhelp import gen, normal

pytestmark = pytest.mark.gpu


def _expert_mul(t, e, i, o):
    import stade_hip as hip
    g = gen(t)
    x, w = (normal(g, *s, dtype=torch.bfloat16).cuda() for s in ((t, i), (e, i, o)))
    y = torch.zeros(t, o, dtype=torch.bfloat16, device="cuda")
    start = (torch.arange(e + 1) * t // e).cuda()
    return lambda: hip.expert_mul(y, x, w, start, i, o, t, e), [y]


def _expert_mul_b(t, e, i, o):
    import stade_hip as hip
    g = gen(t)
    x, w, yb = (normal(g, *s).cuda() for s in ((t, i), (e, i, o), (t, o)))
    xb, wb = torch.zeros(t, i, device="cuda"), torch.zeros(e, i, o, device="cuda")
    start = (torch.arange(e + 1) * t // e).cuda()
    return lambda: hip.expert_mul_b(yb, x, xb, w, wb, start, i, o, t, e, add=False), [xb, wb]


def _embed_b(t, d, v):
    import stade_hip as hip
    g = gen(t)
    yb, tok, wb = normal(g, t, d).cuda(), torch.randint(0, v + 1, (t,), generator=g).cuda(), torch.zeros(v, d, device="cuda")
    return lambda: hip.embed_b(yb, wb, tok, 0.5, d, v, t, add=False), [wb]


def _layernorm_b(n, d):
    import stade_hip as hip
    g = gen(n)
    x, yb, xb = normal(g, n, d).cuda(), normal(g, n, d).cuda(), torch.zeros(n, d, device="cuda")
    gb, bb, mu, rs = torch.zeros(d, device="cuda"), torch.zeros(d, device="cuda"), torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
    return lambda: hip.layernorm_b(yb, x, xb, None, gb, bb, mu, rs, d, n, add=False), [xb, gb, bb]


# function, the largest call, and smaller ones that take more scratch
CASES = {
    "expert_mul": (_expert_mul, (8192, 4, 2048, 2560), [(64, 4, 1672, 2484), (30, 2, 2000, 72)]),
    "expert_mul_b": (_expert_mul_b, (4096, 4, 2048, 2560), [(64, 4, 1672, 2484), (3584, 2, 128, 295)]),
    "embed_b": (_embed_b, (40000, 512, 300), [(32000, 512, 300), (32767, 500, 299)]),
    "layernorm_b": (_layernorm_b, (520, 70000), [(520, 65536), (512, 65537)]),
}


def capture_after_largest(name):
    import stade_hip
    make, largest, smaller = CASES[name]
    print(f"{name}: eager {largest}", flush=True)
    make(*largest)[0]()
    torch.cuda.synchronize()
    for size in smaller:
        call, outs = make(*size)
        print(f"{name}: captured {size}, {stade_hip.workspace_info()[0]} bytes held", flush=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        call()
        torch.cuda.synchronize()
        eager = [v.clone() for v in outs]
        for rep in range(3):
            for v in outs:
                v.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(v, w) for v, w in zip(outs, eager)), f"{name} {size}: replay {rep}"
            _ = torch.randn(1000, device="cuda").sum().item()
    print("captured", flush=True)


def refused_call_enqueues_nothing():
    """Captured with no eager call before: refused, and the graph holds no part of the call."""
    import stade_hip
    call, (xb, wb) = _expert_mul_b(3584, 2, 128, 295)   # (wb in slices, xb not)
    print("expert_mul_b captured first", flush=True)
    stade_hip.workspace_info()   # (the workspace is there, without scratch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(stade_hip.StadeHipError, match="cannot grow under graph capture"):
        with torch.cuda.graph(graph):
            xb.add_(1.0)
            call()
    graph.replay()
    torch.cuda.synchronize()
    assert xb.eq(1.0).all() and not wb.any()
    print("captured", flush=True)


def first_call_without_workspace():
    """Calls that use nothing of the library's are captured with no call before them."""
    import stade_hip as hip
    n, d = 8, 256
    g = gen(5)
    x, yb = normal(g, n, d).cuda(), normal(g, n, d).cuda()
    y, xb, back, wb = (torch.full((n, d), 7.0, device="cuda") for _ in range(4))
    mu, rs, gb, bb = (torch.zeros(k, device="cuda") for k in (n, n, d, d))
    q, qs = torch.zeros(n * d, dtype=torch.int8, device="cuda"), torch.zeros(n * d // 32, dtype=torch.uint8, device="cuda")
    none, no_rows = torch.empty(0, dtype=torch.int64, device="cuda"), torch.empty(0, d, device="cuda")

    def calls():
        hip.layernorm(y, x, None, None, mu, rs, d, n, tape=(q, qs))
        hip.tape8_store(x, q, qs, d, n)
        hip.tape8_load(q, qs, back, d, n)
        hip.layernorm_b(yb, x, xb, None, gb, bb, mu, rs, d, n, add=False)
        hip.embed_b(no_rows, wb, none, 1.0, d, n, 0, add=False)

    print("norms and tape captured first", flush=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    outs = [y, xb, back, wb, mu, rs, gb, bb, q, qs]
    calls()
    torch.cuda.synchronize()
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
            f"import test_gpu_lm_capture as m; m.{call}")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100, cwd=str(ROOT))
    assert r.returncode == 0 and "captured" in r.stdout.split(), r.stdout[-2000:] + r.stderr[-2000:]


def test_a_refused_call_enqueues_nothing():
    print("capture without an eager call: expert_mul_b", flush=True)
    _in_a_process("refused_call_enqueues_nothing()")


def test_first_calls_that_need_no_workspace():
    print("capture without an eager call: norms, tape", flush=True)
    _in_a_process("first_call_without_workspace()")


@pytest.mark.parametrize("name", CASES)
def test_smaller_calls_are_captured_after_the_largest(name):
    print(f"capture after the largest call: {name}", flush=True)
    _in_a_process(f"capture_after_largest({name!r})")
