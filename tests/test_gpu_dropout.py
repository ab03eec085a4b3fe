"""dropout and dropout_b: the mask against the generator written out in whole numbers, the values against
the formula in 64 bits."""
import numpy as np
import pytest
import torch

from lmhelp import IDS, TYPES, U, apart, gen, normal, within


def philox(counter, key):
    """Philox 4x32 with ten rounds of an array (n, 4) of counters, by Python's whole numbers in numpy's 64 bits."""
    c = [np.asarray(counter[:, i], dtype=np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    low, word = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> word) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> word) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack(c, 1).astype(np.uint32)


def mask(key, p, n, d):
    seed, call = (int(v) % 2 ** 64 for v in key)
    m = (d + 7) // 8
    c = np.zeros((n * m, 4), dtype=np.uint64)
    c[:, 0], c[:, 1] = np.tile(np.arange(m), n), np.repeat(np.arange(n), m)
    c[:, 2], c[:, 3] = call % 2 ** 32, call >> 32
    bits = philox(c, (seed % 2 ** 32, seed >> 32)).astype("<u4").view("<u2").reshape(n, 8 * m)[:, :d]
    return torch.from_numpy(bits.astype(np.int64) >= round(65536 * p))


def test_generator_against_its_published_answers():
    """The known answers that were published with the generator (zeros; ones; digits of pi)."""
    ones = 0xFFFFFFFF
    for counter, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((ones,) * 4, (ones,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(v) for v in philox(np.array([counter], dtype=np.uint64), key)[0]) == want


SIZES = [(1, 1), (3, 7), (2, 8), (5, 9), (17, 64), (9, 1001), (300, 515), (1, 20000), (2000, 40)]
KEYS = [(0, 0), (-1, -1), (2 ** 62 + 12345, 7), (-(2 ** 63), 2 ** 40 + 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.99])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_both_sweeps(size, dt, p):
    import stade_hip
    n, d = size
    g = gen(n + d)
    x, r, yb, base = (normal(g, n, d, dtype=dt) for _ in range(4))
    key = KEYS[(n + d) % 4]
    k = torch.tensor(key).cuda()
    keep = mask(key, p, n, d)
    scale = 65536.0 / (65536 - round(65536 * p))
    print(f"dropout {size} {IDS[dt]} p={p}", flush=True)
    y, alone, xb, added = (torch.full_like(x, float("nan")).cuda() for _ in range(4))
    stade_hip.dropout(y, x.cuda(), r.cuda(), k, p, d, n)
    stade_hip.dropout(alone, x.cuda(), None, k, p, d, n)
    stade_hip.dropout_b(yb.cuda(), xb, k, p, d, n, add=False)
    stade_hip.dropout_b(yb.cuda(), added.copy_(base), k, p, d, n)
    zero = torch.zeros((), dtype=torch.float64)
    v, vb = (torch.where(keep, w.double() * scale, zero) for w in (x, yb))
    # the factor, the product and the sum are rounded once each
    within("y", y, r.double() + v, 3 * U * (r.double().abs() + v.abs()), dt)
    within("without a residual", alone, v, 2 * U * v.abs(), dt)
    within("xb", xb, vb, 2 * U * vb.abs(), dt)
    within("xb added", added, base.double() + vb, 3 * U * (base.double().abs() + vb.abs()), dt)
    assert torch.equal(alone.cpu() != 0, keep & (x != 0))
    # rows apart and in place: the same bits
    yv, rv = apart(torch.zeros_like(y)), apart(r.cuda())
    stade_hip.dropout(yv, apart(x.cuda()), rv, k, p, d, n)
    assert torch.equal(yv, y)
    stade_hip.dropout(rv, apart(x.cuda()), rv, k, p, d, n)
    assert torch.equal(rv, y)
    stade_hip.dropout(yv.copy_(x.cuda()), yv, r.cuda(), k, p, d, n)
    assert torch.equal(yv, y)


@pytest.mark.gpu
def test_dropped_values_leave_nothing():
    import stade_hip
    n, d, p = 8, 100, 0.5
    key = torch.tensor([5, 6])
    keep = mask(key.tolist(), p, n, d)
    x = torch.full((n, d), float("nan"))
    x[:, 50:] = float("inf")
    x[keep] = 1.0
    y = torch.empty(n, d, device="cuda")
    stade_hip.dropout(y, x.cuda(), None, key.cuda(), p, d, n)
    assert torch.equal(y.cpu(), torch.where(keep, 2.0, 0.0))


@pytest.mark.gpu
def test_masks_of_calls_differ_and_a_graph_moves_on():
    """The key is read on the device: a captured call takes another mask after the key has moved."""
    import stade_hip
    n, d, p = 64, 256, 0.25
    x, key = torch.ones(n, d, device="cuda"), torch.tensor([11, 0], device="cuda")
    y = torch.empty_like(x)
    stade_hip.dropout(y, x, None, key, p, d, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        key[1:].add_(1)
        stade_hip.dropout(y, x, None, key, p, d, n)
    seen = []
    for call in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu() != 0, mask((11, call), p, n, d))
        seen.append(y.clone())
        _ = torch.randn(1000, device="cuda").sum().item()
    assert not torch.equal(seen[0], seen[1])


@pytest.mark.gpu
def test_share_of_values_that_stay():
    """Of 2^22 values a share within five standard deviations of 1 - p."""
    import stade_hip
    n, d, p = 1024, 4096, 0.3
    x, y = torch.ones(n, d, device="cuda"), torch.empty(n, d, device="cuda")
    stade_hip.dropout(y, x, None, torch.tensor([1, 2], device="cuda"), p, d, n)
    share = y.ne(0).double().mean().item()
    q = 1 - round(65536 * p) / 65536
    assert abs(share - q) <= 5 * (q * (1 - q) / (n * d)) ** 0.5
