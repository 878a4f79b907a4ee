"""The microscaled operators as programs use them: copies and files of their objects, memory between
steps."""
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


def test_backward_frees_the_checkpoints():
    """A training step keeps 33/32 byte a value between its passes, and nothing of it when it is over, with the
    loss still held."""
    from vorotracing_b200 import mx

    rows, cols = 4096, 256
    z = values(rows, cols, torch.bfloat16, scale=1.0).requires_grad_()
    w = values(64, cols, torch.bfloat16, 1, 0.1).requires_grad_()
    mx.act_linear(z, w, None, "silu").float().square().sum().backward()  # what libraries keep from their first call on
    z.grad = w.grad = None
    before = torch.cuda.memory_allocated()
    y = mx.act_linear(z, w, None, "silu")
    kept = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert rows * cols * 33 // 32 <= kept < rows * cols * 33 // 32 + 1024
    loss = y.float().square().sum()
    del y
    loss.backward()
    assert torch.cuda.memory_allocated() - before < (rows * cols + 64 * cols) * 2 + 4096 and loss.isfinite()
