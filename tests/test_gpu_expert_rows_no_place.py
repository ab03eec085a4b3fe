"""Slots without a place beside rows that are not finite: their weights' shadows are 0, or what they were."""
import pytest
import torch

from lmhelp import IDS, TYPES, gen, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dt", TYPES, ids=IDS.get)
@pytest.mark.parametrize("k", [1, 2, 7])
def test_shadows_of_weights(k, dt, bad):
    import stade_hip
    t, d = 9, 70
    place = torch.arange(1, t * k + 1).view(t, k)
    place[2] = place[5, 0] = place[7, k - 1] = 0
    yb, ys, pb0 = normal(gen(1), t, d, dtype=dt), normal(gen(2), t * k, d, dtype=dt), normal(gen(3), t, k)
    p = torch.rand(t, k, generator=gen(4))
    yb[2:8, 33] = bad
    for add in (False, True):
        pb, ysb = pb0.cuda(), torch.zeros(t * k, d, dtype=dt, device="cuda")
        print(f"slots without a place: {k} {IDS[dt]} {bad} {add}", flush=True)
        stade_hip.expert_join_b(yb.cuda(), ys.cuda(), ysb, p.cuda(), pb, place.cuda(), d, k, t, add=add)
        got, none = pb.cpu(), place == 0
        assert torch.equal(got[none], pb0[none] if add else torch.zeros(int(none.sum())))
        rest = ~none
        assert not torch.isfinite(got[2:8][rest[2:8]]).any()
        clean = rest.clone()
        clean[2:8] = False
        assert torch.isfinite(got[clean]).all()
        assert torch.isfinite(ysb.view(t, k, d).cpu()[torch.isfinite(yb).all(1)]).all()
        y = torch.zeros(t, d, dtype=dt, device="cuda")
        stade_hip.expert_join(y, ys.cuda(), p.cuda(), place.cuda(), d, k, t)
        assert torch.isfinite(y).all()
