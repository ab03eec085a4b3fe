"""The 8-bit tape against its definition in 64 bits: equal, value by value."""
import pytest
import torch

from lmhelp import IDS, TYPES, apart, gen, new_tape, normal, tape_values

pytestmark = pytest.mark.gpu


def _round_trip(x, d, n):
    import stade_hip
    q, qs = new_tape(d, n)
    stade_hip.tape8_store(x, q, qs, d, n)
    back = torch.full((n, d), 5.0, dtype=x.dtype, device="cuda")
    stade_hip.tape8_load(q, qs, back, d, n)
    return q, qs, back


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("size", [(1, 1), (1, 31), (3, 32), (2, 33), (7, 100), (129, 515), (1000, 64)], ids=str)
def test_round_trip(size, dt):
    n, d = size
    g = gen(n + d)
    x = (torch.randn(n, d, generator=g) * torch.exp(2 * torch.randn(n, 1, generator=g))).to(dt)
    print(f"tape8 n={n} d={d} {IDS[dt]}", flush=True)
    q, qs, back = _round_trip(x.cuda(), d, n)
    assert torch.equal(back.double().cpu(), tape_values(x.double()))
    assert not q.view(n, -1)[:, d:].any()
    v = apart(x.cuda())
    q2, qs2, back2 = _round_trip(v, d, n)
    assert torch.equal(q, q2) and torch.equal(qs, qs2) and torch.equal(back, back2)


def test_special_values():
    """Zeros, scales at a power of two and on both sides of the step at 127, the ends of the
    exponent range, infinities and NaN (the group, and no other, reads back as NaN)."""
    rows = torch.zeros(12, 64)
    rows[1, 0] = 127.0
    rows[2, 0] = 127.00001
    rows[3, 0], rows[3, 1] = 128.0, 1.0
    rows[4, :32] = torch.linspace(-1, 1, 32)
    rows[5, 3] = 2.0 ** -126
    rows[6, 3] = 1e-42
    rows[7, 3] = float("inf")
    rows[8, 40] = float("nan")
    rows[9, 5], rows[9, 6] = -float("inf"), float("nan")
    rows[10, 0], rows[10, 1] = -127.5, 0.5
    rows[11, 0] = 1.5 * 2.0 ** 127
    print("tape8 special values", flush=True)
    _, qs, back = _round_trip(rows.cuda(), 64, 12)
    want = tape_values(rows.double())
    got = back.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(), want.nan_to_num())
    assert got[8, :32].eq(0).all() and torch.isnan(got[8, 32:]).all() and qs.view(12, 2)[0, 0] == 1


@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
def test_largest_values_stay_finite(dt):
    big = torch.finfo(dt).max
    x = torch.tensor([[big, -big] + [big / 3] * 30], dtype=dt)
    _, _, back = _round_trip(x.cuda(), 32, 1)
    assert torch.isfinite(back).all()
    assert ((back.double().cpu() - x.double()).abs() <= big / 127 * 2).all()


def test_nothing():
    import stade_hip
    assert stade_hip.tape8_lengths(33, 5) == (64 * 5, 2 * 5)
    e = torch.empty(0, device="cuda")
    stade_hip.tape8_store(e, e.to(torch.int8), e.to(torch.uint8), 0, 4)
    stade_hip.tape8_load(e.to(torch.int8), e.to(torch.uint8), e, 4, 0)
