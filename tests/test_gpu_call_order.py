"""Calls of the language-model operators on different streams, with no wait by the caller: a call
on another stream than the previous call's runs behind it, as for every entry point.

The first call's stream is kept busy for some milliseconds before it, so that a second call that did
not wait would read what was there before, or overwrite what the first has yet to read."""
import subprocess
import sys

import pytest
import torch

from lmhelp import gen, new_tape, normal

pytestmark = pytest.mark.gpu

T, D = 48, 256


def _busy(work):
    for _ in range(8):
        torch.mm(work, work)


class Pairs:
    """(first call, second call, what the second leaves): each pair on arrays of its own."""

    def __init__(self):
        import stade_hip as hip
        g = gen(11)
        mat = lambda: normal(g, T, D).cuda()   # noqa: E731
        old = lambda: torch.full((T, D), 7.0, device="cuda")   # noqa: E731
        ids = torch.randperm(T, generator=g).cuda() + 1
        none = torch.empty(0, dtype=torch.int64, device="cuda")
        one, stat = torch.ones(D, device="cuda"), lambda: torch.full((T,), 0.5, device="cuda")   # noqa: E731
        start = torch.tensor([0, 20, T], device="cuda")
        w = normal(g, 2, D, D).cuda()
        x, yb = mat(), mat()
        take = lambda dst, src: hip.embed(dst, src, ids, 1.0, D, T, T)   # noqa: E731
        self.pairs = {}

        a, b = old(), old()
        self.pairs["embed, expert_mul"] = (lambda: take(a, x), lambda: hip.expert_mul(b, a, w, start, D, D, T, 2), b)
        c, d = old(), old()
        self.pairs["layernorm, embed"] = (lambda: hip.layernorm(c, x, one, one, None, None, D, T), lambda: take(d, c), d)
        e, f, mu, rs = old(), old(), stat(), stat()
        self.pairs["layernorm_b of few rows, embed"] = (
            lambda: hip.layernorm_b(yb[:8], x[:8], e[:8], None, None, None, mu[:8], rs[:8], D, 8, add=False), lambda: take(f, e), f)
        h, i = old(), old()
        gb, bb = torch.zeros(D, device="cuda"), torch.zeros(D, device="cuda")
        self.pairs["layernorm_b of many rows, embed"] = (
            lambda: hip.layernorm_b(yb, x, h, None, gb, bb, mu, rs, D, T, add=False), lambda: take(i, h), i)
        tape, j = new_tape(D, T), old()
        hip.tape8_store(old(), *tape, D, T)
        self.pairs["tape8_store, tape8_load"] = (lambda: hip.tape8_store(x, *tape, D, T), lambda: hip.tape8_load(*tape, j, D, T), j)
        held, k, m = new_tape(D, T), old(), old()
        hip.tape8_store(x, *held, D, T)
        self.pairs["tape8_load, embed"] = (lambda: hip.tape8_load(*held, k, D, T), lambda: take(m, k), m)
        n, o = old(), old()
        self.pairs["embed_b of no tokens, embed"] = (
            lambda: hip.embed_b(torch.empty(0, D, device="cuda"), n, none, 1.0, D, T, 0, add=False), lambda: take(o, n), o)
        p, q = x.clone(), new_tape(D, T)
        self.pairs["tape8_store reads, embed overwrites"] = (lambda: hip.tape8_store(p, *q, D, T), lambda: take(p, yb), q[0])
        torch.cuda.synchronize()


def _in_order(first_stream, second_stream, names=None):
    """Every pair on the two streams, against the same pair on one."""
    work = torch.randn(4096, 4096, device="cuda")
    want = {}
    alone = Pairs()
    for name, (first, second, out) in alone.pairs.items():
        first()
        second()
        torch.cuda.synchronize()
        want[name] = out.clone()
    both = Pairs()
    for name in names or both.pairs:
        first, second, out = both.pairs[name]
        print(f"calls in order: {name}", flush=True)
        with torch.cuda.stream(first_stream):
            _busy(work)
            first()
        with torch.cuda.stream(second_stream):
            second()
        torch.cuda.synchronize()
        assert torch.equal(out, want[name]), name


def test_side_stream_first():
    _in_order(torch.cuda.Stream(), torch.cuda.default_stream())


def test_default_stream_first():
    _in_order(torch.cuda.default_stream(), torch.cuda.Stream())


def test_two_side_streams():
    _in_order(torch.cuda.Stream(), torch.cuda.Stream())


def first_of_a_process():
    """The first call ever on a second stream, right behind a call on the default one."""
    _in_order(torch.cuda.default_stream(), torch.cuda.Stream(), ["embed, expert_mul"])
    print("in order", flush=True)


def test_first_second_stream_of_a_process():
    from helpers import ROOT
    code = (f"import sys; sys.path[:0] = [{str(ROOT / 'tests')!r}, {str(ROOT / 'stade.jl_amd')!r}]; "
            "import test_gpu_call_order as m; m.first_of_a_process()")
    print("the first call on a second stream of a process", flush=True)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100, cwd=str(ROOT))
    assert r.returncode == 0 and "in order" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
