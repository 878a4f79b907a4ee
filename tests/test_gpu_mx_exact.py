"""Products of whole numbers, whose sums are exact in binary32 whatever their order: results are the exact sums
rounded once, so that one lost or repeated tile, stage or part of k shows in thousands of elements.

Sums stay below 2^24: rows (or columns) times the largest product.  8-bit blocks hold whole numbers up to 127, 4-bit
blocks -3 to 3."""
import pytest
import torch

from test_gpu_mx import TYPES16, no_kernel_gave_up  # noqa: F401

pytestmark = pytest.mark.gpu


def whole(rows, cols, most, seed, dtype=torch.float64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, (rows, cols), generator=g, device="cuda").to(dtype)


LINEAR = [(60001, 64, 3), (60001, 40, 64), (60000, 16, 16), (60000, 56, 250), (30011, 256, 256), (30011, 200, 130), (30000, 136, 70), (30000, 96, 192),
          (177, 64, 64), (20011, 520, 300), (30001, 48, 427), (3001, 96, 5000), (9001, 777, 1301), (100000, 8, 8), (200000, 130, 1), (150001, 24, 260)]


@pytest.mark.parametrize("act", ["identity", "relu"])
@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("rows,cols,outs", LINEAR)
def test_gradients_of_whole_numbers(rows, cols, outs, dtype, act):
    from vorotracing_b200 import mx

    z, dy, w = whole(rows, cols, 2, 0), whole(rows, outs, 1, 1), whole(outs, cols, 2, 2)
    z[:, 0] = 2  # no block is all zeros
    dy[rows // 3] = 0
    _, ckpt = mx.act_checkpoint(z.to(dtype), act)
    assert torch.equal(ckpt.dequantize().double(), z)
    h, slope = (z.clamp(min=0), (z > 0).double()) if act == "relu" else (z, 1.0)
    got = mx.linear_backward(dy.to(dtype), w.to(dtype), ckpt)
    for name, a, b in zip(("dz", "dw", "db"), got, ((dy @ w) * slope, dy.t() @ h, dy.sum(0))):
        b = b.to(dtype)
        assert torch.equal(a, b), f"{name}: {int((a != b).sum())} of {b.numel()} differ"


LINEAR4 = [(1, 4096, 4096), (77, 1000, 333), (500, 2000, 1000), (60001, 192, 64), (60001, 96, 48), (41000, 300, 100), (41000, 600, 256), (40961, 40, 130),
           (20001, 520, 600), (9601, 91, 195), (2049, 4100, 1300), (100000, 64, 3), (5000, 2056, 449)]


@pytest.mark.parametrize("dtype", TYPES16)
@pytest.mark.parametrize("rows,cols,outs", LINEAR4)
def test_4_bit_products_of_whole_numbers(rows, cols, outs, dtype):
    from vorotracing_b200 import mx

    x, w, b = whole(rows, cols, 3, 0), whole(outs, cols, 3, 1), whole(1, outs, 3, 2)[0]
    w4 = mx.quantize4(w.float())
    assert torch.equal(w4.dequantize().double(), w) and torch.equal(mx.quantize4(x.to(dtype)).dequantize().double(), x)
    for act in ("identity", "relu"):
        got = mx.linear4(x.to(dtype), w4, b.to(dtype), act)
        want = x @ w.t() + b
        want = (want.clamp(min=0) if act == "relu" else want).to(dtype)
        assert torch.equal(got, want), f"{int((got != want).sum())} of {want.numel()} differ"


@pytest.mark.parametrize("rows,cols,outs", [(153512, 16, 224), (200003, 33, 256), (153512, 96, 200), (60001, 300, 250), (153512, 16, 192), (200003, 16, 128), (200003, 8, 8)])
def test_gradients_come_out_the_same_each_time(rows, cols, outs):
    """Many tiles a block whose stores are slow against its products, and many calls: what depends on timing shows."""
    from vorotracing_b200 import mx

    z, dy, w = (whole(*s, 1, i, torch.float16) for i, s in enumerate(((rows, cols), (rows, outs), (outs, cols))))
    _, ckpt = mx.act_checkpoint(z, "identity")
    z8 = ckpt.dequantize().double()
    want = [t.half() for t in (dy.double() @ w.double(), dy.double().t() @ z8, dy.double().sum(0))]
    for _ in range(60):
        for a, b in zip(mx.linear_backward(dy, w, ckpt), want):
            assert torch.equal(a, b)
    mx.raise_errors()
