"""embed_b added to what is there, at row lengths whose last vector shares values with the one before, in all
types: small whole numbers, so every sum is exact and a value added twice, or not at all, shows."""
import pytest
import torch

from lmhelp import IDS, TYPES, apart, gen

pytestmark = pytest.mark.gpu


# few tokens; by counting; sorted in one block; by the radix sort (runs in a chunk and over many)
@pytest.mark.parametrize("t,v", [(60, 7), (3000, 700), (9001, 2500), (20000, 9000)], ids=str)
@pytest.mark.parametrize("d", [9, 15, 33, 127, 513, 515, 519, 520, 777])
@pytest.mark.parametrize("tw", TYPES, ids=IDS.get)
@pytest.mark.parametrize("ty", TYPES, ids=IDS.get)
def test_added_exactly(ty, tw, d, t, v):
    import stade_hip
    g = gen(t + d)
    tok = torch.randint(0, v + 1, (t,), generator=g)
    tok[:40] = 1 + v // 2
    # (no more than 256 in sum, the largest whole number up to which bf16 holds all: one row in ten counts)
    yb = torch.randint(-2, 3, (t, d), generator=g) * (torch.rand(t, 1, generator=g) < 0.1)
    base = torch.randint(-20, 21, (v, d), generator=g)
    want = base.clone().index_add_(0, tok[tok > 0] - 1, yb[tok > 0])
    assert want.abs().max() <= 256
    print(f"embed_b added t={t} v={v} d={d} {IDS[ty]} into {IDS[tw]}", flush=True)
    wb = base.to(tw).cuda()
    stade_hip.embed_b(yb.to(ty).cuda(), wb, tok.cuda(), 1.0, d, v, t)
    assert torch.equal(wb.cpu(), want.to(tw))
    wv = apart(base.to(tw).cuda())
    stade_hip.embed_b(apart(yb.to(ty).cuda()), wv, tok.cuda(), 1.0, d, v, t)
    assert torch.equal(wv, wb)
