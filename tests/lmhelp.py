"""Shared by the tests of the language-model operators: inputs, references in 64 bits, and the
bounds that the operators' arithmetic gives.

Bounds are elementwise.  U is fp32's unit roundoff: an fp32 sum whose additions are nested at
most k deep is within k U of the sum of the terms' absolute values (to first order; the few ulp of
the terms themselves are counted into k).  A result rounded to type T moves by at most
ROUND[T] of its size (half the spacing; for f16 also by half the least subnormal)."""
import torch

U = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def cuda(t):
    return None if t is None else t.cuda()


def apart(t, gap=3):
    """A copy of a matrix whose rows lie `gap` elements further apart, at an odd offset."""
    n, d = t.shape
    big = torch.full((n * (d + gap) + 1,), float("nan") if t.is_floating_point() else 7, dtype=t.dtype, device=t.device)
    v = big[1:].view(n, d + gap)[:, :d]
    v.copy_(t)
    return v


def within(name, got, want, slack, dtype):
    """|got - want| <= slack + what rounding `want` to dtype may add, elementwise; NaN where NaN."""
    got, want, slack = got.detach().double().cpu(), want.double().cpu(), slack.double().cpu()
    assert got.shape == want.shape, f"{name}: shape {tuple(got.shape)} != {tuple(want.shape)}"
    if got.numel() == 0:
        return
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN in other places"
    bound = slack + ROUND[dtype] * (want.abs() + slack) + LEAST[dtype]
    off = (got - want).abs()
    bad = ~(off <= bound) & ~torch.isnan(want) & (got != want)
    if bad.any():
        at = int(bad.flatten().nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {at}: "
                             f"{got.flatten()[at]:.9g}, expected {want.flatten()[at]:.9g} within {bound.flatten()[at]:.3g}")


def tape_values(x):
    """What the 8-bit tape of x (float64) holds: groups of 32 of a row, the least power of two
    2^e with max|x| <= 127 2^e (e >= -126), whole numbers to nearest even."""
    n, d = x.shape
    out = torch.zeros_like(x)
    for j in range(0, d, 32):
        part = x[:, j:j + 32]
        big = part.abs().amax(1)
        ok = torch.isfinite(part).all(1)
        safe = torch.where(ok, big, torch.ones_like(big))
        m, k = torch.frexp(safe)          # safe = m 2^k, 1/2 <= m < 1: 127 2^e >= safe for e = k - 7 up to m = 127/128
        e = torch.where(m > 127.0 / 128.0, k - 6, k - 7)
        e = torch.where(safe == 0, torch.full_like(e, -126), e).clamp_min(-126)
        unit = torch.ldexp(torch.ones_like(safe), e)[:, None]
        out[:, j:j + 32] = torch.where(ok[:, None], torch.round(part / unit) * unit, torch.full_like(part, float("nan")))
    return out


def new_tape(d, n):
    import stade_hip
    lq, ls = stade_hip.tape8_lengths(d, n)
    return torch.full((lq,), 99, dtype=torch.int8, device="cuda"), torch.full((ls,), 99, dtype=torch.uint8, device="cuda")
