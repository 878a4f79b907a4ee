"""The microscaled formats and the operators on them in 64 bits, for the tests.

Written from the formats' definition (include/vorotracing_b200.h), without the
package."""
import math

import torch

BLOCK = 32
# half the spacing of a type's numbers next to 1, and half its smallest spacing
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def blocks_of(x):
    cols = x.size(1)
    pad = -cols % BLOCK
    return torch.nn.functional.pad(x.double(), (0, pad)).view(x.size(0), -1, BLOCK)


def exponent(x, lower, least):
    """floor(log2 max|x|) - lower of each block, at least `least`; and whether the block is finite."""
    top = blocks_of(x).abs().amax(dim=2)
    finite = blocks_of(x).isfinite().all(dim=2)
    _, e = torch.frexp(torch.where(finite, top, torch.ones_like(top)))
    e = torch.where(top == 0, torch.full_like(e, -5000), e - 1 - lower)
    return e.clamp(min=least), finite


def round8(x):
    """(values, codes, exponent bytes) of the 8-bit format."""
    e, finite = exponent(x, 0, -120)
    unit = torch.exp2((e - 6).double()).unsqueeze(2)
    code = torch.round(blocks_of(x) / unit).clamp(-127, 127)
    code = torch.where(finite.unsqueeze(2), code, torch.zeros_like(code))
    v = torch.where(finite.unsqueeze(2), code * unit, torch.full_like(code, math.nan))
    E = torch.where(finite, e + 127, torch.full_like(e, 255))
    return (v.flatten(1)[:, :x.size(1)], code.flatten(1).to(torch.int8), E.to(torch.uint8))


E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def round4(x):
    """(values, exponent bytes) of the 4-bit format: the nearest of the eight magnitudes, the one
    with the even index where two are as near."""
    e, finite = exponent(x, 2, -126)
    unit = torch.exp2(e.double()).unsqueeze(2)
    m = (blocks_of(x) / unit).abs().clamp(max=6)
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    i = torch.bucketize(m, grid).clamp(max=7)      # first magnitude not below m
    j = (i - 1).clamp(min=0)
    up, down = grid[i] - m, m - grid[j]
    pick = torch.where((up < down) | ((up == down) & (i % 2 == 0)), i, j)
    v = grid[pick] * unit * torch.sign(blocks_of(x))
    v = torch.where(finite.unsqueeze(2), v, torch.full_like(v, math.nan))
    E = torch.where(finite, e + 127, torch.full_like(e, 255))
    return v.flatten(1)[:, :x.size(1)], E.to(torch.uint8)


def act(z, name):
    z = z.double()
    if name == "identity":
        return z
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "silu":
        return z * torch.special.expit(z)
    k = math.sqrt(2 / math.pi)
    return z * torch.special.expit(2 * k * (z + 0.044715 * z ** 3))


def slope(z, name):
    z = z.double()
    if name == "identity":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).double()
    if name == "silu":
        p = torch.special.expit(z)
        return p + z * p * torch.special.expit(-z)
    u = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    du = 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2)
    p = torch.special.expit(u)
    return p + z * p * torch.special.expit(-u) * du


def assert_within(got, want, bound, name=""):
    """Every element of `got` within `bound` of `want` (all in 64 bits); equal non-finite places."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.equal(got.isfinite(), want.isfinite()), f"{name}: other places are finite"
    fine = want.isfinite()
    off = (got - want).abs() - torch.broadcast_to(bound, want.shape)
    bad = (off > 0) & fine
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} beyond the bound, first at "
                           f"{bad.nonzero()[0].tolist()}: {got[bad][0].item()} for "
                           f"{want[bad][0].item()}")
