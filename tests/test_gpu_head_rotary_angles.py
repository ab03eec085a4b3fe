"""Angles next to half and quarter turns, where a sine or cosine is small: to Float32's relative accuracy."""
import math

import pytest
import torch

from lmhelp import U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pos", [1, 3, 5, 1001])
@pytest.mark.parametrize("half", [True, False], ids=["half", "neighbours"])
def test_small_sines_and_cosines(half, pos):
    import stade_hip
    r = 128
    off = torch.logspace(-7, -2, r // 2, dtype=torch.float64) * torch.tensor([1.0, -1.0], dtype=torch.float64).repeat(r // 4)
    for quarters in (1, 2, 3):
        freq = (quarters * math.pi / 2 * (1 + off)) / pos
        angle = pos * freq
        x = torch.zeros(1, r)
        if half:
            x[0, r // 2:] = 1         # (a, b) = (0, 1): -sin and cos
        else:
            x[0, 1::2] = 1
        at = torch.tensor([pos]).cuda()
        y = torch.empty(1, r, device="cuda")
        stade_hip.head_rotary(y, x.cuda(), None, None, at, freq.cuda(), r, 1, 0, r, 1, norm=False, half=half)
        back = torch.empty(1, r, device="cuda")
        stade_hip.head_rotary_b(x.cuda(), None, back, None, None, None, None, at, freq.cuda(), r, 1, 0, r, 1, norm=False, half=half, add=False)
        for got, sign in ((y.cpu().double(), -1), (back.cpu().double(), 1)):
            a, b = (got[0, :r // 2], got[0, r // 2:]) if half else (got[0, 0::2], got[0, 1::2])
            # the function to 4 units of the last place, its correction, the factor and the product: 14 U; the whole angle by three
            # roundings in 64 bits
            for v, want in ((a, sign * torch.sin(angle)), (b, torch.cos(angle))):
                bound = 14 * U * want.abs() + 2.0 ** -51 * angle.abs()
                assert ((v - want).abs() <= bound).all(), ((v - want).abs() / want.abs()).max()
