"""The language-model operators in the forms that only larger calls take: each size below says which
kernels it is for, on a card of 256 compute units."""
import pytest
import torch

from lmhelp import IDS, TYPES, gen, new_tape, normal
from test_gpu_expert_mul import NAME
from test_gpu_expert_mul import test_backward as check_expert_backward
from test_gpu_expert_mul import test_forward as check_expert_forward
from test_gpu_layernorm import test_backward as check_norm_backward

pytestmark = pytest.mark.gpu

H = TYPES[1:]   # the 16-bit types

# Products in tiles of 128 x 128 with straight loads: 16-bit types where 256 x 256 tiles would fill between a quarter
# of the CUs and all of them; fp32 from two of them a CU.  (Contiguous arrays; the same calls on rows that lie apart go
# through registers, in fp32 in tiles of the same size.)
Y16 = [([1300, 0, 701], 3, 64, 4096), ([700, 1291], 0, 72, 4104)]
XB16 = [([1300, 0, 701], 3, 4096, 64), ([700, 1291], 0, 4104, 72)]
WB16 = [([70, 0, 133], 2, 1024, 1536), ([1, 64], 0, 2568, 1160)]
Y32 = [([65] * 40, 7, 32, 4400), ([130, 0] * 20, 0, 36, 4356), ([65] * 40, 7, 33, 4401)]
XB32 = [([65] * 40, 7, 4400, 32), ([130, 0] * 20, 0, 4356, 36), ([65] * 40, 7, 4401, 33)]
WB32 = [([5] * 130, 3, 300, 260), ([0, 9] * 65, 0, 260, 388), ([5] * 130, 3, 299, 257)]


@pytest.mark.parametrize("add", [False, True], ids=["set", "add"])
@pytest.mark.parametrize("size,dt", [(s, t) for s in Y16 for t in H] + [(s, torch.float32) for s in Y32],
                         ids=lambda v: NAME(v) if isinstance(v, tuple) else IDS[v])
def test_products_of_middle_tiles(size, dt, add):
    check_expert_forward(size, dt, add)


@pytest.mark.parametrize("add", [False, True], ids=["set", "add"])
@pytest.mark.parametrize("held", ["x", "tape"])
@pytest.mark.parametrize("size,dt", [(s, t) for s in WB16 for t in H] + [(s, torch.float32) for s in WB32],
                         ids=lambda v: NAME(v) if isinstance(v, tuple) else IDS[v])
def test_weight_shadows_of_middle_tiles(size, dt, held, add):
    check_expert_backward(size, dt, held, add)


@pytest.mark.parametrize("add", [False, True], ids=["set", "add"])
@pytest.mark.parametrize("size,dt", [(s, t) for s in XB16 for t in H] + [(s, torch.float32) for s in XB32],
                         ids=lambda v: NAME(v) if isinstance(v, tuple) else IDS[v])
def test_row_shadows_of_middle_tiles(size, dt, add):
    check_expert_backward(size, dt, "x", add)


# rows that the reverse sweep reads again for their sums, more of them than its 512 blocks: a block adds a second row to
# its partial sums
@pytest.mark.parametrize("add", [False, True], ids=["set", "add"])
@pytest.mark.parametrize("tape", [False, True], ids=["x", "tape"])
@pytest.mark.parametrize("size,dt", [((600, 16392), torch.float32), ((530, 16387), torch.bfloat16)], ids=str)
def test_norm_adjoint_of_many_long_rows(size, dt, tape, add):
    check_norm_backward(size, dt, tape, add)


# more rows than the launches have blocks for at once: the same bits as in two calls
def _halves(n):
    return (slice(0, n // 2), slice(n // 2, n))


def test_embed_of_more_rows_than_blocks():
    import stade_hip
    t, d, v = 300001, 8, 5000
    g = gen(1)
    w, tok = normal(g, v, d).cuda(), torch.randint(0, v + 1, (t,), generator=g).cuda()
    print(f"embed t={t}", flush=True)
    y, z = torch.empty(t, d, device="cuda"), torch.empty(t, d, device="cuda")
    stade_hip.embed(y, w, tok, 0.5, d, v, t)
    for r in _halves(t):
        stade_hip.embed(z[r], w, tok[r], 0.5, d, v, r.stop - r.start)
    assert torch.equal(y, z)
    assert torch.equal(y, 0.5 * torch.cat([torch.zeros(1, d, device="cuda"), w])[tok])   # (an exact product)


def test_norm_of_more_rows_than_blocks():
    import stade_hip
    n, d = 270001, 16
    x = torch.randn(n, d, device="cuda")
    print(f"layernorm n={n}", flush=True)
    y, z = torch.empty_like(x), torch.empty_like(x)
    tapes = [new_tape(d, n) for _ in range(2)]
    stade_hip.layernorm(y, x, None, None, None, None, d, n, tape=tapes[0])
    for r in _halves(n):
        part = tuple(v.view(n, -1)[r] for v in tapes[1])
        stade_hip.layernorm(z[r], x[r], None, None, None, None, d, r.stop - r.start, tape=part)
    assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip(*tapes))


def test_tape_of_more_groups_than_blocks():
    import stade_hip
    n, d = 2100001, 33
    x = torch.randn(n, d, device="cuda", dtype=torch.bfloat16)
    print(f"tape8 n={n}", flush=True)
    tapes = [new_tape(d, n) for _ in range(2)]
    back, again = torch.empty_like(x), torch.empty_like(x)
    stade_hip.tape8_store(x, *tapes[0], d, n)
    stade_hip.tape8_load(*tapes[0], back, d, n)
    for r in _halves(n):
        part = tuple(v.view(n, -1)[r] for v in tapes[1])
        stade_hip.tape8_store(x[r], *part, d, r.stop - r.start)
        stade_hip.tape8_load(*part, again[r], d, r.stop - r.start)
    assert all(torch.equal(a, b) for a, b in zip(*tapes)) and torch.equal(back, again)
    assert ((back.float() - x.float()).abs().amax(1) <= x.float().abs().amax(1) / 127).all()


def test_zero_rows_of_more_ids_than_blocks():
    import stade_hip
    v, d = 300001, 5
    wb = torch.ones(v, d, device="cuda")
    print(f"embed_b of no tokens v={v}", flush=True)
    stade_hip.embed_b(torch.empty(0, d, device="cuda"), wb, torch.empty(0, dtype=torch.int64, device="cuda"), 1.0, d, v, 0, add=False)
    assert not wb.any()
