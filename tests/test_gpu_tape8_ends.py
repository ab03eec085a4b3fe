"""The 8-bit tape's bound at both ends of the exponent range: a value reads back within max|x| / 127 of
its group, or within 2^-127 where that is more."""
import pytest
import torch

from lmhelp import IDS, TYPES, gen, new_tape

pytestmark = pytest.mark.gpu


def _stored(x, how):
    """x's values as its tape holds them, written by tape8_store or by layernorm."""
    import stade_hip
    n, d = x.shape
    x, tape = x.cuda(), new_tape(d, n)
    if how == "store":
        stade_hip.tape8_store(x, *tape, d, n)
    else:
        stade_hip.layernorm(torch.empty_like(x), x, None, None, None, None, d, n, tape=tape)
    back = torch.full_like(x, 5.0)
    stade_hip.tape8_load(*tape, back, d, n)
    return back.double().cpu()


def _bound(x):
    big = x.double().abs().unflatten(1, (-1, 32)).amax(2, keepdim=True).expand(-1, -1, 32).flatten(1)
    return (big / 127.0).clamp_min(2.0 ** -127)


@pytest.mark.parametrize("how", ["store", "layernorm"])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
def test_largest_values(dt, how):
    """Groups whose largest value is one of the type's last, on both sides of 127/128 of the next power of two."""
    top = torch.finfo(dt).max
    x = (torch.rand(40, 64, generator=gen(1), dtype=torch.float64) * 2 - 1) * top
    for row in range(40):   # (the last 2 % of the range, and the largest value itself)
        x[row, row % 32], x[row, 32 + row % 32] = top * (1 - 0.0005 * row), -top
    x = x.to(dt)
    assert torch.isfinite(x).all()
    print(f"tape8 largest values {IDS[dt]} {how}", flush=True)
    back = _stored(x, how)
    assert torch.isfinite(back).all()
    assert ((back - x.double()).abs() <= _bound(x)).all()


@pytest.mark.parametrize("how", ["store", "layernorm"])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=IDS.get)
def test_least_values(dt, how):
    """Groups at and below the least scale: whole numbers of 2^-126, to nearest even."""
    x = torch.zeros(6, 32, dtype=torch.float64)
    x[0, :4] = torch.tensor([0.75, 0.5, -1.5, 2.5]) * 2.0 ** -126
    x[1, 0], x[1, 1] = 2.0 ** -127, -(2.0 ** -133)
    x[2, 0], x[2, 1] = 127 * 2.0 ** -126, 2.0 ** -126
    x[3, 0], x[3, 1] = 128 * 2.0 ** -126, 2.0 ** -126
    x[4] = torch.linspace(-1, 1, 32, dtype=torch.float64) * 2.0 ** -125
    x[5] = torch.linspace(-1, 1, 32, dtype=torch.float64) * 2.0 ** -119
    x = x.to(dt)
    print(f"tape8 least values {IDS[dt]} {how}", flush=True)
    back = _stored(x, how)
    assert ((back - x.double()).abs() <= _bound(x)).all()
    assert (back[0, :4] * 2.0 ** 126).tolist() == [1.0, 0.0, -2.0, 2.0] and not back[1].any()
