"""Infinities in upstream gradients, as a loss scale that is too large makes them: they spread as far as the
formulas say and no further."""
import pytest
import torch

import mx_reference as R
from test_gpu_mx import TYPES16, no_kernel_gave_up  # noqa: F401

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
