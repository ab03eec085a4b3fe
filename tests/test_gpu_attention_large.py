"""The operators around attention and the experts on arrays of more than 2^31 elements: the rows at the end, whose offsets do not fit
32 bits, against calls on those rows alone (the same bits)."""
import pytest
import torch

from test_gpu_dropout import philox
from test_gpu_lm_large import BF, D, LAST, N, _free, _rows   # noqa: F401 (_free: after each test)

pytestmark = pytest.mark.gpu
H, HEAD = 8, 128        # N * H * HEAD = 2^31 + 3.8e4


def test_attention_of_many_sequences():
    import stade_hip as hip
    q, k, v, yb = (_rows(N, H * HEAD) for _ in range(4))
    k.mul_(0.5)
    start = torch.cat([torch.arange(0, N - LAST, 1000), torch.tensor([N - LAST, N])]).cuda()
    last = slice(N - LAST, N)

    def run(q, k, v, yb, start):
        t, n = q.shape[0], len(start) - 1
        y, lse = torch.empty_like(q), torch.empty(t, H, device="cuda")
        qb, kb, vb = (torch.empty_like(a) for a in (q, k, v))
        size = (HEAD, H, H, t, t, n)
        # (a window in which no tile's rows go over several blocks)
        hip.attention(y, lse, q, k, v, start, start, 0.1, *size, window=30, check=True)
        hip.attention_b(yb, y, lse, q, qb, k, kb, v, vb, start, start, 0.1, *size, window=30, add=False, check=True)
        return [a[-LAST:].clone() for a in (y, lse, qb, kb, vb)]
    print("attention: 2^31 values each", flush=True)
    got = run(q, k, v, yb, start)
    want = run(*(a[last].clone() for a in (q, k, v, yb)), torch.tensor([0, LAST]).cuda())
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_one_token_of_a_long_cache():
    """Single tokens whose keys lie past 2^31 elements of the cache."""
    import stade_hip as hip
    k, v = _rows(N, H * HEAD), _rows(N, H * HEAD)
    q = _rows(2, H * HEAD)
    far = N - 7000
    print("attention: a cache of 2^31 values", flush=True)

    def run(k, v, at):
        y, lse = torch.empty_like(q), torch.empty(2, H, device="cuda")
        hip.attention(y, lse, q, k, v, torch.tensor([0, 1, 2]).cuda(), torch.tensor(at).cuda(), 0.1, HEAD, H, H, 2, k.shape[0], 2, check=True)
        return y, lse
    y, lse = run(k, v, [far, far + 3000, N])
    q32, c = q.double().view(2, H, HEAD), 0.1
    for i, (a, b) in enumerate(((far, far + 3000), (far + 3000, N))):
        kk, vv = k[a:b].double().view(-1, H, HEAD), v[a:b].double().view(-1, H, HEAD)
        s = c * (kk * q32[i]).sum(2)
        p = s.softmax(0)
        want = (p[..., None] * vv).sum(0).view(-1)
        # the weights' rounding to bf16, all of one sign, and the result's
        bound = 2.0 ** -8 * ((p[..., None] * vv.abs()).sum(0).view(-1) + 2 * want.abs()) + 1e-4
        assert ((y[i].double() - want).abs() <= bound).all()
        assert ((lse[i].double() - s.logsumexp(0)).abs() <= 1e-3).all()


def test_heads_turned():
    import stade_hip as hip
    x, yb = _rows(N, H * HEAD), _rows(N, H * HEAD)
    pos, freq, g = torch.arange(N, device="cuda"), torch.from_numpy(hip.rotary_freq(HEAD)).cuda(), torch.ones(HEAD, device="cuda")
    print("head_rotary: 2^31 values", flush=True)
    y, xb, gb = torch.empty_like(x), torch.empty_like(x), torch.zeros(HEAD, device="cuda")
    hip.head_rotary(y, x, g, g, pos, freq, HEAD, 5, 3, HEAD, N)
    hip.head_rotary_b(yb, x, xb, g, gb, g, None, pos, freq, HEAD, 5, 3, HEAD, N, add=False)
    a, b = (torch.empty(LAST, H * HEAD, dtype=BF, device="cuda") for _ in range(2))
    hip.head_rotary(a, x[-LAST:], g, g, pos[-LAST:].clone(), freq, HEAD, 5, 3, HEAD, LAST)
    hip.head_rotary_b(yb[-LAST:], x[-LAST:], b, g, None, g, None, pos[-LAST:].clone(), freq, HEAD, 5, 3, HEAD, LAST, add=False)
    assert torch.equal(y[-LAST:], a) and torch.equal(xb[-LAST:], b) and torch.isfinite(gb).all()


def test_rows_to_experts_and_back():
    import stade_hip as hip
    x = _rows(N, D)
    place = (N - torch.arange(N, device="cuda"))[:, None].contiguous()      # the last row first
    p = torch.rand(N, 1, device="cuda")
    print("expert rows: 2^31 values", flush=True)
    xs = torch.empty_like(x)
    hip.expert_take(xs, x, place, D, 1, N, check=True)
    assert torch.equal(xs[:LAST], x[-LAST:].flip(0)) and torch.equal(xs[-LAST:], x[:LAST].flip(0))
    y = torch.empty_like(x)
    hip.expert_join(y, xs, p, place, D, 1, N, check=True)
    for rows in (slice(0, LAST), slice(N - LAST, N)):
        assert torch.equal(y[rows], (p[rows] * x[rows].float()).to(BF))
    pb = torch.empty(N, 1, device="cuda")
    hip.expert_join_b(x, xs, y, p, pb, place, D, 1, N, add=False, check=True)
    assert torch.equal(y[:LAST], (p[-LAST:] * x[-LAST:].float()).to(BF).flip(0))
    want = (x[-LAST:].double() ** 2).sum(1)
    assert ((pb[-LAST:, 0].double() - want).abs() <= 1100 * 2.0 ** -24 * want).all()


def test_dropped():
    import numpy as np
    import stade_hip as hip
    x = _rows(N, D)
    y = torch.empty_like(x)
    print("dropout: 2^31 values", flush=True)
    hip.dropout(y, x, None, torch.tensor([5, 6]).cuda(), 0.5, D, N)
    c = np.zeros((LAST * D // 8, 4), dtype=np.uint64)
    c[:, 0], c[:, 1], c[:, 2] = np.tile(np.arange(D // 8), LAST), np.repeat(np.arange(N - LAST, N), D // 8), 6
    keep = torch.from_numpy(philox(c, (5, 0)).astype("<u4").view("<u2").reshape(LAST, D).astype(np.int64) >= 32768).cuda()
    assert torch.equal(y[-LAST:], torch.where(keep, 2 * x[-LAST:], torch.zeros_like(x[-LAST:])))
