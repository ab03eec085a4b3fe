"""The language-model operators on arrays of more than 2^31 elements: the rows at the end, whose offsets do not
fit 32 bits, against calls on those rows alone (the same bits)."""
import pytest
import torch

from lmhelp import new_tape

pytestmark = pytest.mark.gpu

N, D, LAST = (1 << 21) + 37, 1032, 50   # N * D = 2^31 + 1.7e7
BF = torch.bfloat16


def _rows(n, d):
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    x = torch.empty(n, d, dtype=BF, device="cuda")
    x.normal_(generator=g)
    return x


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def test_token_rows():
    import stade_hip as hip
    w = _rows(N, D)
    tok = torch.tensor([N, 1, N - 1, 0, N - 20, N], device="cuda")
    print("embed, embed_b: a table of 2^31 values", flush=True)
    y = torch.empty(6, D, dtype=BF, device="cuda")
    hip.embed(y, w, tok, 1.0, D, N, 6, check=True)
    want = w[(tok - 1).clamp_min(0)]
    want[3] = 0
    assert torch.equal(y, want)
    # as many rows out of a small table
    back = torch.full_like(w, 5.0)
    ids = torch.randint(0, LAST + 1, (N,), device="cuda")
    hip.embed(back, w[:LAST], ids, 1.0, D, LAST, N)
    tail = torch.empty(LAST, D, dtype=BF, device="cuda")
    hip.embed(tail, w[:LAST], ids[-LAST:], 1.0, D, LAST, LAST)
    assert torch.equal(back[-LAST:], tail)
    del back
    wb = torch.full_like(w, 5.0)
    hip.embed_b(y, wb, tok, 1.0, D, N, 6, add=False)
    assert torch.equal(wb[N - 1], (y[0].float() + y[5].float()).to(BF)) and torch.equal(wb[N - 2], y[2]) and torch.equal(wb[N - 21], y[4])
    assert torch.equal(wb[0], y[1]) and not wb[N - 20:N - 2].any() and not wb[1:9].any()


def test_many_rows_summed():
    import stade_hip as hip
    yb = _rows(N, D)
    tok = torch.ones(N, dtype=torch.int64, device="cuda")
    tok[-LAST:] = torch.arange(2, LAST + 2, device="cuda")
    print("embed_b: 2^31 values of shadows", flush=True)
    wb = torch.empty(LAST + 1, D, device="cuda")
    hip.embed_b(yb, wb, tok, 1.0, D, LAST + 1, N, add=False)
    assert torch.equal(wb[1:], yb[-LAST:].float())


def test_norm_and_tape():
    import stade_hip as hip
    x, one = _rows(N, D), torch.ones(D, device="cuda")
    mu, rs = torch.empty(N, device="cuda"), torch.empty(N, device="cuda")
    print("layernorm, tape8: 2^31 values", flush=True)
    y, tape = torch.empty_like(x), new_tape(D, N)
    hip.layernorm(y, x, one, one, mu, rs, D, N, tape=tape)
    end, held = slice(N - LAST, N), new_tape(D, LAST)
    z = torch.empty(LAST, D, dtype=BF, device="cuda")
    hip.layernorm(z, x[end], one, one, None, None, D, LAST, tape=held)
    assert torch.equal(y[end], z)
    assert all(torch.equal(a.view(N, -1)[end], b.view(LAST, -1)) for a, b in zip(tape, held))
    other = new_tape(D, N)
    hip.tape8_store(x, *other, D, N)
    assert all(torch.equal(a, b) for a, b in zip(tape, other))
    hip.tape8_load(*tape, y, D, N)
    hip.tape8_load(*held, z, D, LAST)
    assert torch.equal(y[end], z)
    # the reverse sweep, from x and from the tape
    for src, sub in ((dict(x=x), dict(x=x[end])), (dict(x=None, tape=tape), dict(x=None, tape=held))):
        xb, gb, bb = torch.empty_like(x), torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
        hip.layernorm_b(x, src["x"], xb, one, gb, bb, mu, rs, D, N, add=False, tape=src.get("tape"))
        hip.layernorm_b(x[end], sub["x"], z, one, None, None, mu[end], rs[end], D, LAST, add=False, tape=sub.get("tape"))
        assert torch.equal(xb[end], z)
        del xb


@pytest.mark.parametrize("aligned", [True, False], ids=["straight", "through registers"])
def test_products_of_many_rows(aligned):
    import stade_hip as hip
    d = D if aligned else D + 1
    x, o = _rows(N, d), 64
    w = _rows(2 * d, o).view(2, d, o)
    start = torch.tensor([0, N - LAST, N], device="cuda")
    end, last = slice(N - LAST, N), torch.tensor([0, 0, LAST], device="cuda")
    print(f"expert_mul, expert_mul_b: 2^31 values of rows, aligned={aligned}", flush=True)
    y, z = torch.empty(N, o, dtype=BF, device="cuda"), torch.empty(LAST, o, dtype=BF, device="cuda")
    hip.expert_mul(y, x, w, start, d, o, N, 2, check=True)
    near = lambda a, b: ((a.float() - b).abs() <= 0.02 * b.abs().max()).all()   # noqa: E731
    assert near(y[end], x[end].float() @ w[1].float())
    xb, wb = torch.empty_like(x), torch.empty(2, d, o, device="cuda")
    hip.expert_mul_b(y, x, xb, w, wb, start, d, o, N, 2, add=False, check=True)
    assert near(xb[end], y[end].float() @ w[1].float().t().contiguous())
    assert near(wb[1], x[end].float().t().contiguous() @ y[end].float())
    wl = torch.empty(2, d, o, device="cuda")
    hip.expert_mul_b(y[end], x[end], None, None, wl, last, d, o, LAST, 2, add=False)
    assert near(wb[1], wl[1])
    tape, held = new_tape(d, N), new_tape(d, LAST)
    hip.tape8_store(x, *tape, d, N)
    hip.tape8_store(x[end], *held, d, LAST)
    hip.expert_mul_b(y, None, None, None, wb, start, d, o, N, 2, add=False, tape=tape)
    hip.expert_mul_b(y[end], None, None, None, wl, last, d, o, LAST, 2, add=False, tape=held)
    assert near(wb[1], wl[1])


def test_products_of_many_weights():
    import stade_hip as hip
    e, i, o = 520, 2048, 2056   # 2.19e9 weights
    w = _rows(e * i, o).view(e, i, o)
    t = 2 * e
    start = torch.arange(e + 1, device="cuda") * 2
    x, yb = _rows(t, i), _rows(t, o)
    print("expert_mul, expert_mul_b: 2^31 weights", flush=True)
    y, xb, wb = torch.empty(t, o, dtype=BF, device="cuda"), torch.empty(t, i, dtype=BF, device="cuda"), torch.full_like(w, 5.0)
    hip.expert_mul(y, x, w, start, i, o, t, e, check=True)
    hip.expert_mul_b(yb, x, xb, w, wb, start, i, o, t, e, add=False, check=True)
    near = lambda a, b: ((a.float() - b).abs() <= 0.02 * b.abs().max()).all()   # noqa: E731
    for k in (0, e - 12, e - 1):
        r = slice(2 * k, 2 * k + 2)
        assert near(y[r], x[r].float() @ w[k].float())
        assert near(xb[r], yb[r].float() @ w[k].float().t().contiguous())
        assert near(wb[k], x[r].float().t().contiguous() @ yb[r].float())
