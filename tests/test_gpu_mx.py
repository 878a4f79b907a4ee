"""Microscaled operators against their definition in 64 bits.

Bounds.  u is half the spacing of the output type next to 1 (one rounding of the
result).  A sum of n terms in binary32, in any order and with truncating adders,
is within n 2^-23 of the sum of the terms' magnitudes.  An activation or its
slope in binary32 is within 2^-19 (1 + |z|) of the exact one: the exponential's
argument has a relative error of a few 2^-24 and a magnitude below 90 where the
result is not negligible.  The activations that enter dW are rounded to the
operands' type: u of each term more."""
import pytest
import torch

import mx_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_kernel_gave_up():
    yield
    from vorotracing_b200 import mx

    mx.raise_errors()

TYPES = [torch.float32, torch.float16, torch.bfloat16]
TYPES16 = [torch.float16, torch.bfloat16]
ACTS = ["identity", "relu", "silu", "gelu_tanh"]


def values(rows, cols, dtype, seed=0, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, cols), generator=g, device="cuda") * scale
    x *= torch.exp2(torch.randint(-6, 3, (rows, 1), generator=g, device="cuda").float())
    return x.to(dtype)


def special(dtype):
    """Rows with zeros, ties, the type's extremes, infinities and NaN."""
    x = torch.zeros((12, 70), device="cuda")
    x[1] = torch.linspace(-2, 2, 70, device="cuda")
    x[2, :8] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    x[3, :8] = -x[2, :8]
    x[4, 40] = float("inf")
    x[5, 69] = float("nan")
    x[6, 0] = float("-inf")
    x[7] = torch.finfo(dtype).max
    x[8] = torch.finfo(dtype).tiny
    x[9, ::2] = -0.0
    x[10] = 127.49
    x[11] = 2.0 ** -20
    x = x.to(dtype)
    x[8, 1::3] = torch.finfo(dtype).smallest_normal / 8
    x[11, 3] = 1.0
    return x


SHAPES = [(1, 1), (1, 32), (3, 31), (5, 33), (2, 64), (7, 193), (129, 100), (1000, 8)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_formats_hold_the_definition(rows, cols, dtype):
    from vorotracing_b200 import mx

    x = values(rows, cols, dtype)
    h, ckpt = mx.act_checkpoint(x, "identity")
    v, codes, exps = R.round8(x)
    assert torch.equal(h, x)
    assert torch.equal(ckpt.codes, codes) and torch.equal(ckpt.exps, exps)
    assert torch.equal(ckpt.dequantize().double(), v)
    v, exps = R.round4(x)
    q = mx.quantize4(x)
    assert torch.equal(q.exps, exps) and q.codes.shape == (rows, -(-cols // 32) * 16)
    assert torch.equal(q.dequantize().double(), v)
    for t in TYPES16:
        assert torch.equal(q.dequantize(t), v.to(t)) and torch.equal(ckpt.dequantize(t), R.round8(x)[0].to(t))


@pytest.mark.parametrize("dtype", TYPES)
def test_formats_on_special_values(dtype):
    from vorotracing_b200 import mx

    x = special(dtype)
    v, codes, exps = R.round8(x)
    _, ckpt = mx.act_checkpoint(x, "identity")
    assert torch.equal(ckpt.codes, codes) and torch.equal(ckpt.exps, exps)
    torch.testing.assert_close(ckpt.dequantize().double(), v, rtol=0, atol=0, equal_nan=True)
    v, exps = R.round4(x)
    q = mx.quantize4(x)
    assert torch.equal(q.exps, exps)
    torch.testing.assert_close(q.dequantize().double(), v, rtol=0, atol=0, equal_nan=True)


def act_bound(z):
    return 2.0 ** -19 * (1 + z.double().abs())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (7, 193), (65, 64)])
def test_activation_and_its_gradient(rows, cols, act, dtype):
    from vorotracing_b200 import mx

    z, dh = values(rows, cols, dtype), values(rows, cols, dtype, seed=1)
    h, ckpt = mx.act_checkpoint(z, act)
    u, tiny = R.UNIT[dtype], R.TINY[dtype]
    want = R.act(z, act)
    R.assert_within(h, want, u * want.abs() + act_bound(z) + tiny, "h")
    z8 = R.round8(z)[0]
    want = dh.double() * R.slope(z8, act)
    dz = mx.act_backward(dh, ckpt)
    assert dz.dtype == dtype and dz.shape == dh.shape
    R.assert_within(dz, want, u * want.abs() + dh.double().abs() * act_bound(z8) + tiny, "dz")


@pytest.mark.parametrize("act", ACTS)
def test_activation_gradient_against_differences(act):
    """Central differences of the activation in 64 bits at the 8-bit values.  Their own error is
    step^2 / 6 times the third derivative (below 5 for all) plus 2^-52 |z| / step."""
    from vorotracing_b200 import mx

    z = values(64, 96, torch.float32, seed=3, scale=1.0)
    _, ckpt = mx.act_checkpoint(z, act)
    z8 = ckpt.dequantize().double()
    step = 2.0 ** -14
    want = (R.act(z8 + step, act) - R.act(z8 - step, act)) / (2 * step)
    if act == "relu":  # no derivative at the bend
        want[z8.abs() <= step] = R.slope(z8, act)[z8.abs() <= step]
    got = mx.act_backward(torch.ones_like(z), ckpt)
    R.assert_within(got, want, step ** 2 + 2.0 ** -36 + act_bound(z8), "dz")


def test_activation_passes_infinities_and_nan_on():
    from vorotracing_b200 import mx

    z = torch.zeros((2, 64), device="cuda")
    z[0, 3], z[0, 40], z[1, 5] = float("nan"), float("inf"), -1e30
    for act in ("relu", "silu", "gelu_tanh"):
        h, ckpt = mx.act_checkpoint(z, act)
        assert h[0, 3].isnan() and h[0, 40].isposinf() and h[1, 5] == 0
        dz = mx.act_backward(torch.ones_like(z), ckpt)
        assert dz[0].isnan().all()           # both blocks of the row hold one
        assert dz[1].isfinite().all()


LINEAR = [(1, 1, 1), (1, 32, 8), (5, 33, 3), (64, 64, 64), (77, 200, 31), (128, 96, 130),
          (257, 256, 72), (300, 520, 264), (1000, 64, 3), (4099, 40, 16)]


def linear_want(dy, w, z8, act):
    """(value, sum of the terms' magnitudes) of dz, dW and db, in 64 bits."""
    dy, w = dy.double(), w.double()
    h, s = R.act(z8, act), R.slope(z8, act)
    return {"dz": ((dy @ w) * s, (dy.abs() @ w.abs()), s),
            "dw": (dy.t() @ h, dy.t().abs() @ h.abs()),
            "db": (dy.sum(0), dy.abs().sum(0))}


def check_linear(got, dy, w, z8, act):
    rows, outs = dy.shape
    dtype = dy.dtype
    u, tiny = R.UNIT[dtype], R.TINY[dtype]
    want = linear_want(dy, w, z8, act)
    v, size, s = want["dz"]
    R.assert_within(got[0], v, u * v.abs() + size * (outs * 2.0 ** -23 * s.abs() + act_bound(z8)) + tiny, "dz")
    v, size = want["dw"]
    extra = dy.double().abs().t() @ (act_bound(z8) + tiny)
    R.assert_within(got[1], v, u * v.abs() + (u * (1 + u) + rows * 2.0 ** -23) * size + extra + tiny, "dw")
    v, size = want["db"]
    R.assert_within(got[2], v, u * v.abs() + rows * 2.0 ** -23 * size + tiny, "db")


# several tiles for every SM
LINEAR += [(60001, 64, 3), (60001, 40, 64), (60000, 56, 250), (30011, 256, 256), (30011, 200, 130), (30000, 136, 70), (30000, 96, 192),
           (20011, 520, 300), (3001, 96, 5000)]


@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("rows,cols,outs", LINEAR)
def test_linear_backward(rows, cols, outs, dtype):
    from vorotracing_b200 import mx

    act = ACTS[(rows + cols + outs) % 4]
    z = values(rows, cols, dtype, scale=1.0)
    dy, w = values(rows, outs, dtype, seed=1, scale=0.5), values(outs, cols, dtype, seed=2, scale=0.3)
    dy[rows // 2] = 0  # a ray behind a mask
    _, ckpt = mx.act_checkpoint(z, act)
    check_linear(mx.linear_backward(dy, w, ckpt), dy, w, R.round8(z)[0], act)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,cols,outs", [(700, 128, 128), (3000, 64, 200)])
def test_linear_backward_activations(rows, cols, outs, act):
    from vorotracing_b200 import mx

    z = values(rows, cols, torch.bfloat16, scale=1.0)
    dy, w = values(rows, outs, torch.bfloat16, 1), values(outs, cols, torch.bfloat16, 2, 0.3)
    _, ckpt = mx.act_checkpoint(z, act)
    check_linear(mx.linear_backward(dy, w, ckpt), dy, w, R.round8(z)[0], act)


@pytest.mark.parametrize("dtype", TYPES16)
def test_linear_backward_strides_and_parts(dtype):
    """Rows of a wider matrix, a start that is not 16-byte aligned, a transposed gradient; outputs
    that were not asked for."""
    from vorotracing_b200 import mx

    rows, cols, outs = 333, 72, 40
    z = values(rows, cols, dtype, scale=1.0)
    _, ckpt = mx.act_checkpoint(z, "silu")
    z8 = R.round8(z)[0]
    dy, w = values(rows, outs, dtype, 1), values(outs, cols, dtype, 2, 0.3)
    wide = values(rows, outs + 24, dtype, 3)
    wide[:, 1:outs + 1] = dy
    wide_w = values(outs, cols + 9, dtype, 4)
    wide_w[:, 3:cols + 3] = w
    whole = mx.linear_backward(dy, w, ckpt)
    check_linear(whole, dy, w, z8, "silu")
    for a, b in ((wide[:, 1:outs + 1], wide_w[:, 3:cols + 3]), (dy.t().contiguous().t(), w.t().contiguous().t())):
        for x, y in zip(mx.linear_backward(a, b, ckpt), whole):
            assert torch.equal(x, y)
    only = mx.linear_backward(dy, w, ckpt, bias=False, need_dw=False)
    assert torch.equal(only[0], whole[0]) and only[1] is None and only[2] is None
    only = mx.linear_backward(dy, w, ckpt, bias=False, need_dz=False)
    assert only[0] is None and torch.equal(only[1], whole[1]) and only[2] is None
    only = mx.linear_backward(dy, w, ckpt, need_dz=False, need_dw=False)
    assert torch.equal(only[2], whole[2])


def test_linear_backward_against_differences():
    """Differences of the loss sum(y * g) in 64 bits along random directions of z, W and b; z holds
    8-bit values already.  Along a direction the outputs' roundings (u each) add up."""
    from vorotracing_b200 import mx

    dtype, act, rows, cols, outs = torch.float16, "silu", 96, 64, 48
    z = R.round8(values(rows, cols, dtype, scale=0.5))[0].to(dtype)
    g, w = values(rows, outs, dtype, 1, 0.2), values(outs, cols, dtype, 2, 0.2)
    _, ckpt = mx.act_checkpoint(z, act)
    assert torch.equal(ckpt.dequantize(dtype), z)
    dz, dw, db = (t.double() for t in mx.linear_backward(g, w, ckpt))
    gen = torch.Generator(device="cuda").manual_seed(9)
    loss = lambda z, w, b: ((R.act(z, act) @ w.t() + b) * g.double()).sum()
    step, u = 2.0 ** -10, R.UNIT[dtype]
    zero = torch.zeros(outs, dtype=torch.float64, device="cuda")
    for i, (x, grad) in enumerate(((z.double(), dz), (w.double(), dw), (zero, db))):
        d = torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float64)
        args = [z.double(), w.double(), zero]
        hi, lo = list(args), list(args)
        hi[i], lo[i] = x + step * d, x - step * d
        want = (loss(*hi) - loss(*lo)) / (2 * step)
        terms = (grad * d).abs().sum()
        # differences: third derivatives below 1 a term, |d| below 6
        slack = 4 * u * terms + step ** 2 * 36 * (g.double().abs() @ w.double().abs()).sum()
        assert (grad * d).sum().sub(want).abs() <= slack


def test_linear_backward_nan_blocks_and_zeros():
    from vorotracing_b200 import mx

    z = values(40, 64, torch.bfloat16, scale=1.0)
    z[7, 40] = float("nan")
    dy, w = values(40, 16, torch.bfloat16, 1), values(16, 64, torch.bfloat16, 2)
    _, ckpt = mx.act_checkpoint(z, "silu")
    dz, dw, db = mx.linear_backward(dy, w, ckpt)
    assert dz[7, 32:].isnan().all() and dz[7, :32].isfinite().all() and dz[8].isfinite().all()
    assert dw[:, 32:].isnan().all() and dw[:, :32].isfinite().all() and db.isfinite().all()
    z.zero_()
    _, ckpt = mx.act_checkpoint(z, "silu")
    dz, dw, _ = mx.linear_backward(dy, w, ckpt)
    assert not dw.any() and dz.isfinite().all()


def test_linear_backward_is_reproducible():
    from vorotracing_b200 import mx

    z, dy, w = values(20000, 64, torch.bfloat16), values(20000, 24, torch.bfloat16, 1), values(24, 64, torch.bfloat16, 2)
    _, ckpt = mx.act_checkpoint(z, "relu")
    first = mx.linear_backward(dy, w, ckpt)
    for _ in range(3):
        for a, b in zip(mx.linear_backward(dy, w, ckpt), first):
            assert torch.equal(a, b)


LINEAR4 = [(1, 1, 1), (1, 64, 8), (1, 4096, 512), (2, 33, 3), (16, 1000, 333), (17, 256, 128), (64, 96, 130),
           (77, 1000, 77), (130, 520, 264), (300, 192, 64), (1000, 75, 48), (513, 1024, 640), (128, 4100, 200),
           (9600, 96, 40), (10000, 75, 8), (9999, 200, 128), (9700, 520, 200), (2000, 333, 1300), (5000, 256, 512)]


# several tiles for every SM, so that stages, accumulators and buffers are used again
LINEAR4 += [(60001, 192, 64), (60001, 96, 48), (41000, 300, 100), (41000, 600, 256), (40960, 40, 130), (20001, 520, 600)]


@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("rows,cols,outs", LINEAR4)
def test_linear4(rows, cols, outs, dtype):
    from vorotracing_b200 import mx

    act = ACTS[(rows + cols + outs) % 4]
    x, w = values(rows, cols, dtype, scale=1.0), values(outs, cols, torch.float32, 1, 0.3)
    b = values(1, outs, dtype, 2)[0] if (rows + outs) % 3 else None
    y = mx.linear4(x, mx.quantize4(w), b, act)
    x4, w4 = R.round4(x)[0], R.round4(w)[0]
    pre = x4 @ w4.t() + (b.double() if b is not None else 0)
    size = x4.abs() @ w4.abs().t() + (b.double().abs() if b is not None else 0)
    want, u = R.act(pre, act), R.UNIT[dtype]
    # no activation is steeper than 1.13
    bound = u * want.abs() + 1.13 * (cols + 1) * 2.0 ** -23 * size + act_bound(pre) + R.TINY[dtype]
    R.assert_within(y, want, bound, "y")


@pytest.mark.parametrize("rows", [1, 3, 40, 300])
def test_linear4_strides_and_special_values(rows):
    from vorotracing_b200 import mx

    w = mx.quantize4(values(48, 90, torch.float32, 1))
    wide = values(rows, 131, torch.bfloat16)
    x = wide[:, 7:97]
    y = mx.linear4(x, w)
    assert torch.equal(y, mx.linear4(x.contiguous(), w))
    assert torch.equal(y, mx.linear4(x.t().contiguous().t(), w))
    assert torch.equal(y.view(1, rows, 48), mx.linear4(x.reshape(1, rows, 90), w))
    x = x.clone()
    x[rows // 2, 50] = float("nan")
    y = mx.linear4(x, w)
    assert y[rows // 2].isnan().all() and y.isfinite().sum() == (rows - 1) * 48
    wide = values(48, 90, torch.float32, 1)
    wide[5, 0] = float("inf")
    y = mx.linear4(x.nan_to_num(), mx.quantize4(wide))
    assert y[:, 5].isnan().all() and y.isfinite().sum() == rows * 47


def test_empty_matrices():
    from vorotracing_b200 import mx

    e = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda")
    h, ckpt = mx.act_checkpoint(e(0, 64))
    assert h.shape == (0, 64) and mx.act_backward(e(0, 64), ckpt).shape == (0, 64)
    dz, dw, db = mx.linear_backward(e(0, 8), e(8, 64), ckpt)
    assert dz.shape == (0, 64) and not dw.any() and not db.any()
    _, ckpt = mx.act_checkpoint(values(5, 64, torch.bfloat16))
    dz, dw, db = mx.linear_backward(e(5, 0), e(0, 64), ckpt)
    assert not dz.any() and dw.shape == (0, 64) and db.shape == (0,)
    _, ckpt = mx.act_checkpoint(e(5, 0))
    dy = torch.ones((5, 3), dtype=torch.bfloat16, device="cuda")
    dz, dw, db = mx.linear_backward(dy, e(3, 0), ckpt)
    assert dz.shape == (5, 0) and dw.shape == (3, 0) and torch.equal(db, torch.full_like(db, 5))
    assert mx.quantize4(e(0, 64)).dequantize().shape == (0, 64)
    w = mx.quantize4(values(3, 64, torch.bfloat16))
    assert mx.linear4(e(0, 64), w).shape == (0, 3)
    assert mx.linear4(e(5, 64), mx.quantize4(e(0, 64))).shape == (5, 0)
    b = torch.tensor([1.0, -2.0, 3.0], device="cuda").bfloat16()
    y = mx.linear4(e(5, 0), mx.quantize4(e(3, 0)), b, "relu")
    assert torch.equal(y, b.clamp(min=0).expand(5, 3))


def test_offsets_past_32_bits():
    """More than 2^32 values: the last rows equal the same rows alone."""
    from vorotracing_b200 import mx

    rows, cols = (1 << 21) + 3, 2056
    z = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    z[-3:] = values(3, cols, torch.bfloat16)
    z[:-3] = 1
    h, ckpt = mx.act_checkpoint(z, "silu")
    h3, c3 = mx.act_checkpoint(z[-3:].clone(), "silu")
    assert torch.equal(h[-3:], h3) and torch.equal(ckpt.codes[-3:], c3.codes) and torch.equal(ckpt.exps[-3:], c3.exps)
    del h
    assert torch.equal(mx.act_backward(z, ckpt)[-3:], mx.act_backward(z[-3:], c3))
    dy, w = values(rows, 8, torch.bfloat16, 1), values(8, cols, torch.bfloat16, 2)
    assert torch.equal(mx.linear_backward(dy, w, ckpt, False, True, False)[0][-3:],
                       mx.linear_backward(dy[-3:], w, c3, False, True, False)[0])
    del ckpt
    w4 = mx.quantize4(values(8, cols, torch.float32, 3))
    assert torch.equal(mx.quantize4(z).codes[-3:], mx.quantize4(z[-3:]).codes)
    assert torch.equal(mx.linear4(z, w4)[-300:], mx.linear4(z[-300:], w4))


def test_side_stream():
    from vorotracing_b200 import mx

    z, dy, w = values(4096, 256, torch.bfloat16), values(4096, 64, torch.bfloat16, 1), values(64, 256, torch.bfloat16, 2)
    _, ckpt = mx.act_checkpoint(z)
    want = (*mx.linear_backward(dy, w, ckpt), mx.linear4(z, mx.quantize4(w)))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(2_000_000)
        late = z * 0 + z                      # written on s behind the sleep
        _, ckpt = mx.act_checkpoint(late)
        got = (*mx.linear_backward(dy, w, ckpt), mx.linear4(late, mx.quantize4(w)))
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_graph_capture():
    from vorotracing_b200 import mx

    z, dy, w = values(300, 128, torch.bfloat16), values(300, 64, torch.bfloat16, 1), values(64, 128, torch.bfloat16, 2)

    def step():
        h, ckpt = mx.act_checkpoint(z)
        return (h, *mx.linear_backward(dy, w, ckpt), mx.linear4(z, mx.quantize4(w)))

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    z.copy_(values(300, 128, torch.bfloat16, 7))
    g.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


def test_act_linear_autograd():
    from vorotracing_b200 import mx

    z, w = values(500, 96, torch.bfloat16, scale=1.0), values(40, 96, torch.bfloat16, 1, 0.2)
    b, g = values(1, 40, torch.bfloat16, 2)[0], values(500, 40, torch.bfloat16, 3)
    for t in (z, w, b):
        t.requires_grad_()
    y = mx.act_linear(z, w, b, "silu")
    h, ckpt = mx.act_checkpoint(z.detach(), "silu")
    assert torch.equal(y, torch.nn.functional.linear(h, w, b))
    y.backward(g)
    for t, want in zip((z, w, b), mx.linear_backward(g, w.detach(), ckpt)):
        assert torch.equal(t.grad, want)
    y = mx.act_linear(z.view(5, 100, 96), w, None, "relu")
    assert y.shape == (5, 100, 40)
    (dz,) = torch.autograd.grad(y, z, g.view(5, 100, 40))
    assert dz.shape == z.shape


def test_refusals():
    from vorotracing_b200 import mx

    z = values(8, 64, torch.bfloat16)
    _, ckpt = mx.act_checkpoint(z)
    w, dy = values(16, 64, torch.bfloat16), values(8, 16, torch.bfloat16)
    w4 = mx.quantize4(w)

    def refused(text, f, *a, **k):
        with pytest.raises(RuntimeError, match=text):
            f(*a, **k)

    refused("CUDA device", mx.act_checkpoint, z.cpu())
    refused("unknown activation", mx.act_checkpoint, z, "tanh")
    refused("dtype float64", mx.act_checkpoint, z.double())
    refused("at least one dimension", mx.act_checkpoint, z[0, 0])
    refused("the checkpoint has 8 of 64", mx.act_backward, z[:, :32], ckpt)
    refused("dtype float32, expected one of float16, bfloat16", mx.linear_backward, dy.float(), w.float(), ckpt)
    refused("dtype of dy", mx.linear_backward, dy, w.half(), ckpt)
    refused("weight had shape", mx.linear_backward, dy, w[:8], ckpt)
    refused("the checkpoint has 8", mx.linear_backward, dy[:4], w, ckpt)
    refused("the checkpoint has 8", mx.linear_backward, dy, w[:, :32], ckpt)
    refused("the weight has 64", mx.linear4, z[:, :32], w4)
    refused("dtype float32, expected", mx.linear4, z.float(), w4)
    refused("bias must have", mx.linear4, z, w4, torch.zeros(16, device="cuda"))
    refused("bias must have", mx.linear4, z, w4, torch.zeros(15, device="cuda").bfloat16())
    refused("unknown activation", mx.linear4, z, w4, None, "gelu")
    refused("take codes", mx.MX4, w4.codes, w4.exps, 65)
    refused("codes must be uint8", mx.MX4, w4.codes.view(torch.int8), w4.exps, 64)
    refused("contiguous", mx.MX4, torch.zeros((16, 16), dtype=torch.uint8, device="cuda").t(),
            torch.zeros((16, 1), dtype=torch.uint8, device="cuda"), 32)
    refused("32-byte aligned", mx.Checkpoint, torch.zeros(8 * 64 + 1, dtype=torch.int8, device="cuda")[1:].view(8, 64),
            ckpt.exps, 64, "relu")
    refused("cannot dequantise", w4.dequantize, torch.float64)


def test_entry_points_refuse():
    """The C entry points check what reaches them themselves."""
    from vorotracing_b200 import mx
    from vorotracing_b200._lib import lib

    z = values(8, 64, torch.bfloat16)
    p = z.data_ptr()
    err = lambda: lib().vt_last_error().decode()
    f = mx._call
    assert f("vt_mx8_checkpoint")(p, 2, 8, 64, 32, 0, p, p, p, None) == 1 and "row stride" in err()
    assert f("vt_mx8_checkpoint")(None, 2, 8, 64, 64, 0, p, p, p, None) == 1 and "null pointer" in err()
    assert f("vt_mx8_checkpoint")(p, 3, 8, 64, 64, 0, p, p, p, None) == 1 and "element type" in err()
    assert f("vt_mx8_checkpoint")(p, 2, 8, 64, 64, 4, p, p, p, None) == 1 and "activation" in err()
    assert f("vt_mx8_act_bwd")(p, 2, 8, 64, 64, p + 8, p, 0, p, None) == 1 and "aligned" in err()
    assert f("vt_mx4_quantize")(p, 2, 8, 64, 64, p, None, None) == 1 and "null pointer" in err()
    assert f("vt_mx4_linear")(p, 64, 2, 10000, 64, 300, p, p, None, 0, p, None, 0, None, None) == 1 and "workspace" in err()
    assert f("vt_mx4_linear")(p, 64, 0, 8, 64, 4, p, p, None, 0, p, p, 1 << 20, None, None) == 1 and "16" in err()
    assert f("vt_mx8_linear_bwd")(p, 4, p, 64, 2, 1 << 32, 64, 4, p, p, 0, p, p, p, p, 1 << 40, None, None) == 1 and "rows" in err()
    assert f("vt_mx8_linear_bwd")(p, 4, None, 64, 2, 8, 64, 4, p, p, 0, p, p, p, p, 1 << 40, None, None) == 1 and "null" in err()


@pytest.mark.parametrize("rows,cols,outs", [(1, 64, 3), (65, 40, 16), (129, 64, 64), (161, 200, 256), (300, 96, 300), (1000, 264, 30)])
def test_linear_backward_writes_its_outputs_only(rows, cols, outs):
    """dz, dW and db in the middle of larger buffers, whose other bytes keep their value."""
    from vorotracing_b200 import mx

    z, dy, w = values(rows, cols, torch.bfloat16), values(rows, outs, torch.bfloat16, 1), values(outs, cols, torch.bfloat16, 2)
    _, ckpt = mx.act_checkpoint(z, "silu")
    want = mx.linear_backward(dy, w, ckpt)
    pads = [torch.full((t.numel() + 131072,), 7.0, dtype=torch.bfloat16, device="cuda") for t in want]
    at = 65536
    p = [t.data_ptr() + 2 * at for t in pads]
    copies = mx._unaligned(dy.data_ptr(), outs) + 2 * mx._unaligned(w.data_ptr(), cols)
    n = mx._call("vt_mx8_linear_bwd_workspace_bytes")(rows, cols, outs, copies)
    ws = torch.full((n + 131072,), 7, dtype=torch.uint8, device="cuda")
    assert mx._call("vt_mx8_linear_bwd")(dy.data_ptr(), outs, w.data_ptr(), cols, 2, rows, cols, outs, ckpt.codes.data_ptr(),
                                         ckpt.exps.data_ptr(), 2, *p, ws.data_ptr() + at, n, None, None) == 0
    torch.cuda.synchronize()
    assert (ws[:at] == 7).all() and (ws[at + n:] == 7).all()
    for t, x in zip(want, pads):
        assert torch.equal(x[at:at + t.numel()].view(t.shape), t)
        assert (x[:at] == 7).all() and (x[at + t.numel():] == 7).all()


@pytest.mark.parametrize("rows,cols,outs", [(1, 64, 3), (77, 1000, 333), (130, 96, 40), (9601, 40, 24), (9601, 96, 200), (1300, 64, 4000)])
def test_linear4_writes_its_output_only(rows, cols, outs):
    from vorotracing_b200 import mx

    x, w = values(rows, cols, torch.float16), mx.quantize4(values(outs, cols, torch.float32, 1))
    want = mx.linear4(x, w)
    at = 65536
    y = torch.full((want.numel() + 2 * at,), 7.0, dtype=torch.float16, device="cuda")
    n = mx._call("vt_mx4_linear_workspace_bytes")(rows, cols, outs, mx._unaligned(x.data_ptr(), cols))
    ws = torch.full((n + 2 * at,), 7, dtype=torch.uint8, device="cuda")
    assert mx._call("vt_mx4_linear")(x.data_ptr(), cols, 1, rows, cols, outs, w.codes.data_ptr(), w.exps.data_ptr(), None, 0,
                                     y.data_ptr() + 2 * at, ws.data_ptr() + at, n, None, None) == 0
    torch.cuda.synchronize()
    assert (ws[:at] == 7).all() and (ws[at + n:] == 7).all()
    assert torch.equal(y[at:at + want.numel()].view(want.shape), want)
    assert (y[:at] == 7).all() and (y[at + want.numel():] == 7).all()
