"""Infinities and NaN in every kernel, and rows with gaps: they spread as far as the
formulas say and no further, and what lies between the rows is not read."""
import pytest
import torch

import mx_reference as R
from test_gpu_mx import TYPES16, no_kernel_gave_up, values  # noqa: F401

pytestmark = pytest.mark.gpu


def same_kind(got, want):
    """Which numbers are NaN, and which infinite with what sign."""
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isposinf(), want.isposinf())
    assert torch.equal(got.isneginf(), want.isneginf())


@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("rows,cols,outs", [(100, 64, 16), (5000, 40, 8), (100, 20, 3), (5001, 64, 70), (5000, 48, 200), (5000, 96, 40), (100, 200, 130),
                                            (3000, 96, 300), (3001, 300, 301)])
def test_infinite_gradients(rows, cols, outs, dtype):
    from vorotracing_b200 import mx

    g = torch.Generator(device="cuda").manual_seed(rows)
    rand = lambda *s: torch.rand(s, generator=g, device="cuda")
    sign = lambda *s: torch.randint(0, 2, s, generator=g, device="cuda") * 2 - 1
    z = ((0.5 + 0.5 * rand(rows, cols)) * sign(rows, cols)).to(dtype)  # no value near zero, whose product with an infinity is a NaN
    w = ((0.5 + 0.5 * rand(outs, cols)) * sign(outs, cols)).to(dtype)
    _, ckpt = mx.act_checkpoint(z, "identity")
    z8 = R.round8(z)[0]
    for row in (0, rows // 2, rows - 1, rows // 2 + 17):
        dy = (0.1 * (rand(rows, outs) - 0.5)).to(dtype)
        dy[row, outs // 2] = float("inf") if row % 2 else float("-inf")
        d = dy.double()
        for got, want in zip(mx.linear_backward(dy, w, ckpt), (d @ w.double(), d.t() @ z8, d.sum(0))):
            assert not want.isnan().any() and want.isinf().any()
            same_kind(got, want)


# linear4: one CTA a tile with x as it is and as a copy, pairs of CTAs with x read in whole words and not, k split
LINEAR4 = [(9700, 90, 48), (9700, 96, 48), (9700, 91, 200), (9700, 96, 256), (5000, 96, 512), (5000, 91, 512), (5000, 300, 449), (100, 600, 200)]


@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("rows,cols,outs", LINEAR4)
def test_nan_and_infinite_blocks_of_4_bits(rows, cols, outs, dtype):
    """A block of x that holds one makes its row NaN, a block of the weight its output; all else keeps its value."""
    from vorotracing_b200 import mx

    x, wide = values(rows, cols, dtype, scale=1.0), values(outs, cols, torch.float32, 1, 0.3)
    w = mx.quantize4(wide)
    want = mx.linear4(x, w)
    assert want.isfinite().all()
    bad = x.clone()
    hit = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for row, col, v in ((0, 0, "nan"), (rows // 2, cols - 1, "inf"), (rows - 1, cols // 2, "-inf"), (rows // 2 + 1, 33, "nan")):
        bad[row, col] = float(v)
        hit[row] = True
    y = mx.linear4(bad, w)
    assert y[hit].isnan().all() and torch.equal(y[~hit], want[~hit])
    out = torch.zeros(outs, dtype=torch.bool, device="cuda")
    for o, col, v in ((0, 1, "inf"), (outs // 2, cols - 1, "nan"), (outs - 1, 32, "-inf")):
        wide[o, col] = float(v)
        out[o] = True
    y = mx.linear4(x, mx.quantize4(wide))
    assert y[:, out].isnan().all() and torch.equal(y[:, ~out], want[:, ~out])


@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("rows,cols,outs", LINEAR4)
def test_4_bit_products_of_rows_with_gaps(rows, cols, outs, dtype):
    from vorotracing_b200 import mx

    x, w = values(rows, cols, dtype, scale=1.0), mx.quantize4(values(outs, cols, torch.float32, 1, 0.3))
    want = mx.linear4(x, w)
    for gap, shift in ((8 + -cols % 8, 0), (8 + -cols % 8, 8), (3, 0), (2, 5), (-cols % 2 + 2, 2)):
        m = torch.full((rows * (cols + gap) + shift,), float("nan"), dtype=dtype, device="cuda")
        v = m[shift:].view(rows, cols + gap)[:, :cols]
        v.copy_(x)
        assert torch.equal(mx.linear4(v, w), want)


LINEAR = [(3000, 96, 300), (3001, 48, 427), (5000, 300, 1000), (3000, 64, 70), (3001, 40, 5), (3000, 200, 256)]


@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("rows,cols,outs", LINEAR)
def test_nan_blocks_of_8_bits(rows, cols, outs, dtype):
    """dz is NaN in the block's own row and columns, dW in its columns; all else keeps its value."""
    from vorotracing_b200 import mx

    for act in ("identity", "relu", "silu", "gelu_tanh"):
        z, dy, w = values(rows, cols, dtype, scale=1.0), values(rows, outs, dtype, 1, 0.5), values(outs, cols, dtype, 2, 0.3)
        _, ckpt = mx.act_checkpoint(z, act)
        want = mx.linear_backward(dy, w, ckpt)
        column = torch.zeros(cols, dtype=torch.bool, device="cuda")
        element = torch.zeros((rows, cols), dtype=torch.bool, device="cuda")
        for row, col, v in ((0, 0, "nan"), (rows - 1, cols - 1, "inf"), (rows // 2, 1, "-inf")):
            z[row, col] = float(v)
            first = col // 32 * 32
            column[first:first + 32] = True
            element[row, first:first + 32] = True
        _, ckpt = mx.act_checkpoint(z, act)
        dz, dw, db = mx.linear_backward(dy, w, ckpt)
        # the slope of the identity is 1 whatever the value
        if act == "identity":
            assert torch.equal(dz[~element], want[0][~element])
        else:
            assert dz[element].isnan().all() and torch.equal(dz[~element], want[0][~element])
        assert dw[:, column].isnan().all() and torch.equal(dw[:, ~column], want[1][:, ~column]) and torch.equal(db, want[2])


def test_every_exponent_of_4_bits():
    """Matrices that were quantised elsewhere: all of a byte's scales, 2^-127 to 2^127."""
    from vorotracing_b200 import mx

    exps = torch.arange(255, device="cuda").to(torch.uint8).view(255, 1)
    codes = torch.arange(16, device="cuda").to(torch.uint8).expand(255, 16).contiguous()  # the even columns: every code
    q = mx.MX4(codes, exps, 32)
    table = torch.tensor([s * v for s in (1, -1) for v in R.E2M1], dtype=torch.float64, device="cuda")
    want = torch.zeros((255, 32), dtype=torch.float64, device="cuda")
    want[:, ::2] = table * torch.exp2(exps.double() - 127)
    got = q.dequantize()
    assert torch.equal(got, want.float()) and got[0, 2] == 2.0 ** -128
    # products of the smallest scales with large values: sums of exact products, 16 terms
    x = torch.full((3, 32), 2.0 ** 100, dtype=torch.bfloat16, device="cuda")
    x[1] = -x[1]
    low = mx.MX4(codes[:4, :].contiguous(), exps[:4].contiguous(), 32)
    low.codes[:, 8:] = 0  # no negatives: 21 units in a row
    want = x.double() @ low.dequantize().double().t()
    assert torch.equal(mx.linear4(x, low), want.bfloat16()) and (want != 0).all()


@pytest.mark.parametrize("outs", [5, 40, 300])
def test_every_exponent_of_8_bits(outs):
    """Checkpoints that were made elsewhere: scales below those that act_checkpoint writes."""
    from vorotracing_b200 import mx

    exps = torch.arange(255, device="cuda").to(torch.uint8).view(255, 1)
    codes = (torch.arange(32, device="cuda") * 8 - 128).to(torch.int8).expand(255, 32).contiguous()
    ckpt = mx.Checkpoint(codes, exps, 32, "identity")
    z8 = codes.double() * torch.exp2(exps.double() - 133)
    z8[254] = z8[254].float().double()  # -128 there is 2^128, an infinity
    assert torch.equal(ckpt.dequantize(), z8.float()) and (ckpt.dequantize()[0, :16] < 0).all()
    # act_backward and the slope of z below zero and above
    ckpt = mx.Checkpoint(codes, exps, 32, "relu")
    dz = mx.act_backward(torch.ones((255, 32), device="cuda"), ckpt)
    assert torch.equal(dz, (z8 > 0).float())
    # the smallest scales alone: dW is the sum of a row's values times a large number
    few = mx.Checkpoint(codes[:8].contiguous(), exps[:8].contiguous(), 32, "identity")
    dy = torch.zeros((8, outs), dtype=torch.bfloat16, device="cuda")
    dy[0], dy[6] = 2.0 ** 100, 2.0 ** 100
    w = torch.ones((outs, 32), dtype=torch.bfloat16, device="cuda")
    dw = mx.linear_backward(dy, w, few)[1]
    want = dy.double().t() @ z8[:8].bfloat16().double()
    assert torch.equal(dw, want.bfloat16()) and (want[:, 20:] > 0).all()
