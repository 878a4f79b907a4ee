"""The microscaled operators as programs use them: copies and files of their objects."""
import copy
import io

import pytest
import torch

from test_gpu_mx import no_kernel_gave_up, values  # noqa: F401

pytestmark = pytest.mark.gpu


def saved(q):
    f = io.BytesIO()
    torch.save(q, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("how", [copy.deepcopy, saved])
def test_a_copied_decoder_has_weights_of_its_own(how):
    from vorotracing_b200.decoder import RayDecoder

    torch.manual_seed(3)
    fast = RayDecoder(features=16, hidden=32).quantized()
    x = values(300, 16, torch.bfloat16)
    want = fast(x)
    other = how(fast)
    for w, b in fast.layers:
        w.codes.zero_(), w.exps.fill_(127), b.zero_()
    assert torch.equal(other(x), want) and not fast(x).any()


@pytest.mark.parametrize("how", [copy.deepcopy, saved])
def test_a_copied_checkpoint_has_codes_of_its_own(how):
    from vorotracing_b200 import mx

    z, dy, w = values(200, 96, torch.bfloat16), values(200, 40, torch.bfloat16, 1), values(40, 96, torch.bfloat16, 2)
    _, ckpt = mx.act_checkpoint(z, "silu")
    want = (mx.act_backward(z, ckpt), *mx.linear_backward(dy, w, ckpt), ckpt.dequantize())
    other = how(ckpt)
    ckpt.codes.zero_(), ckpt.exps.fill_(7)
    got = (mx.act_backward(z, other), *mx.linear_backward(dy, w, other), other.dequantize())
    for a, b in zip(got, want):
        assert torch.equal(a, b)
