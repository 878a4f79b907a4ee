"""Microscaled operators on rows of every alignment: widths that 16, 8 and 4 bytes or only an element
divide, short and long, with strides between the rows, and what lies around the results."""
import pytest
import torch

import mx_reference as R
from test_gpu_mx import ACTS, TYPES, TYPES16, act_bound, check_linear, no_kernel_gave_up, values  # noqa: F401

pytestmark = pytest.mark.gpu

# a row's 9 blocks are the fewest that are read a block at a time; 8 blocks of a warp then cross 0, 1 or more rows
WIDTHS = [2, 3, 4, 6, 12, 30, 34, 36, 63, 255, 257, 258, 260, 287, 289, 319, 515, 1929]


def matrix(rows, cols, dtype, gap, shift, seed=0):
    """A view with `gap` elements between its rows that starts `shift` elements into its memory."""
    m = torch.full((rows * (cols + gap) + shift,), float("nan"), dtype=dtype, device="cuda")
    v = m[shift:].view(rows, cols + gap)[:, :cols]
    v.copy_(values(rows, cols, dtype, seed))
    return v


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gap,shift", [(0, 0), (3, 1), (4, 2)])
@pytest.mark.parametrize("cols", WIDTHS)
def test_formats_at_every_alignment(cols, gap, shift, dtype):
    from vorotracing_b200 import mx

    for rows in (1, 5, 67):
        x = matrix(rows, cols, dtype, gap, shift)
        h, ckpt = mx.act_checkpoint(x, "identity")
        v, codes, exps = R.round8(x)
        assert torch.equal(h, x)
        assert torch.equal(ckpt.codes, codes) and torch.equal(ckpt.exps, exps)
        assert torch.equal(ckpt.dequantize().double(), v)
        v, exps = R.round4(x)
        q = mx.quantize4(x)
        assert torch.equal(q.exps, exps) and torch.equal(q.dequantize().double(), v)
        for t in TYPES16:
            assert torch.equal(q.dequantize(t), v.to(t)) and torch.equal(ckpt.dequantize(t), R.round8(x)[0].to(t))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,gap,shift", [(67, 6, 0, 0), (67, 36, 0, 0), (41, 257, 0, 0), (41, 289, 3, 1), (9, 515, 1, 0), (1001, 300, 2, 2)])
def test_gradient_at_every_alignment(rows, cols, gap, shift, dtype):
    from vorotracing_b200 import mx

    act = ACTS[cols % 4]
    z, dh = matrix(rows, cols, dtype, gap, shift), matrix(rows, cols, dtype, shift, gap, 1)
    h, ckpt = mx.act_checkpoint(z, act)
    u, tiny = R.UNIT[dtype], R.TINY[dtype]
    want = R.act(z, act)
    R.assert_within(h, want, u * want.abs() + act_bound(z) + tiny, "h")
    z8 = R.round8(z)[0]
    want = dh.double() * R.slope(z8, act)
    R.assert_within(mx.act_backward(dh, ckpt), want, u * want.abs() + dh.double().abs() * act_bound(z8) + tiny, "dz")


@pytest.mark.parametrize("dtype,code", list(zip(TYPES, range(3))))
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 36), (3, 257), (67, 289), (9, 515), (33, 256)])
def test_elementwise_write_their_outputs_only(rows, cols, dtype, code):
    from vorotracing_b200 import mx

    at, blocks = 4096, -(-cols // 32)
    x = values(rows, cols, dtype)
    h0, k = mx.act_checkpoint(x, "relu")
    q = mx.quantize4(x)

    def around(n, t):
        return torch.full((n + 2 * at,), 7, dtype=t, device="cuda")

    def check(buf, want):
        n = want.numel()
        assert torch.equal(buf[at:at + n].view(want.shape), want)
        assert (buf[:at] == 7).all() and (buf[at + n:] == 7).all()

    def ptr(buf):
        return buf.data_ptr() + at * buf.element_size()

    n = rows * blocks
    h, codes, exps = around(rows * cols, dtype), around(n * 32, torch.int8), around(n, torch.uint8)
    assert mx._call("vt_mx8_checkpoint")(x.data_ptr(), code, rows, cols, cols, 1, ptr(h), ptr(codes), ptr(exps), None) == 0
    dz, out8, out4 = (around(rows * cols, dtype) for _ in range(3))
    assert mx._call("vt_mx8_act_bwd")(x.data_ptr(), code, rows, cols, cols, ptr(codes), ptr(exps), 1, ptr(dz), None) == 0
    assert mx._call("vt_mx8_dequantize")(ptr(codes), ptr(exps), rows, cols, code, ptr(out8), None) == 0
    codes4, exps4 = around(n * 16, torch.uint8), around(n, torch.uint8)
    assert mx._call("vt_mx4_quantize")(x.data_ptr(), code, rows, cols, cols, ptr(codes4), ptr(exps4), None) == 0
    assert mx._call("vt_mx4_dequantize")(ptr(codes4), ptr(exps4), rows, cols, code, ptr(out4), None) == 0
    torch.cuda.synchronize()
    for buf, want in ((h, h0), (codes, k.codes), (exps, k.exps), (dz, mx.act_backward(x, k)), (out8, k.dequantize(dtype)),
                      (codes4, q.codes), (exps4, q.exps), (out4, q.dequantize(dtype))):
        check(buf, want)


@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("rows,cols,outs", [(1, 33, 257), (31, 48, 300), (300, 50, 300), (129, 1001, 400), (9001, 48, 427), (5000, 45, 259),
                                            (2049, 300, 1025)])
def test_linear_backward_of_unaligned_rows(rows, cols, outs, dtype):
    from vorotracing_b200 import mx

    act = ACTS[(rows + cols) % 4]
    z = values(rows, cols, dtype, scale=1.0)
    dy, w = matrix(rows, outs, dtype, 3, 1, 1), values(outs, cols, dtype, seed=2, scale=0.3)
    _, ckpt = mx.act_checkpoint(z, act)
    check_linear(mx.linear_backward(dy, w, ckpt), dy, w, R.round8(z)[0], act)


@pytest.mark.parametrize("rows,cols,outs", [(31, 48, 300), (129, 1001, 400), (9001, 48, 427)])
def test_linear_backward_of_unaligned_rows_writes_its_outputs_only(rows, cols, outs):
    from test_gpu_mx import test_linear_backward_writes_its_outputs_only

    test_linear_backward_writes_its_outputs_only(rows, cols, outs)


@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("rows,cols,outs", [(127, 91, 195), (9601, 91, 195), (9601, 64, 33), (9700, 96, 127), (4000, 200, 301), (20001, 64, 999)])
def test_linear4_of_unaligned_rows(rows, cols, outs, dtype):
    from test_gpu_mx import test_linear4, test_linear4_writes_its_output_only

    test_linear4(rows, cols, outs, dtype)
    test_linear4_writes_its_output_only(rows, cols, outs)
