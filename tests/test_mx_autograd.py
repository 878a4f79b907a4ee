"""act_linear's autograd function on the host, the kernels behind it replaced by torch operations."""
import weakref

import numpy as np
import pytest
import torch

import mx_reference as R


@pytest.fixture
def mx(monkeypatch):
    from vorotracing_b200 import mx

    def act_checkpoint(z, act="silu"):
        """A checkpoint as the operator makes it, one buffer of codes and exponents, on the host."""
        ckpt = mx.Checkpoint.__new__(mx.Checkpoint)
        ckpt.act, ckpt._act = act, mx.ACTS[act]
        ckpt._new(z, *z.shape)
        memory = np.zeros(ckpt._buf.numel(), np.uint8)
        ckpt._buf = torch.from_numpy(memory)
        mx.kept.append(weakref.ref(memory))
        _, codes, exps = R.round8(z.detach())
        ckpt.codes.copy_(codes)
        ckpt.exps.copy_(exps)
        return R.act(z, act).to(z.dtype), ckpt

    def linear_backward(dy, weight, ckpt, bias=True, need_dz=True, need_dw=True):
        unit = torch.exp2(ckpt.exps.double() - 133).repeat_interleave(32, dim=1)
        z8 = (ckpt.codes.double() * unit)[:, :ckpt.cols]
        g, t = dy.double(), dy.dtype
        return (((g @ weight.double()) * R.slope(z8, ckpt.act)).to(t) if need_dz else None,
                (g.t() @ R.act(z8, ckpt.act)).to(t) if need_dw else None, g.sum(0).to(t) if bias else None)

    monkeypatch.setattr(mx, "kept", [], raising=False)  # memory of the checkpoints made
    monkeypatch.setattr(mx, "act_checkpoint", act_checkpoint)
    monkeypatch.setattr(mx, "linear_backward", linear_backward)
    return mx


def layer(dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(0)
    return [torch.randn(s, generator=g).to(dtype).requires_grad_() for s in ((6, 32), (5, 32), (5,))]


def test_gradients_of_the_first_order(mx):
    z, w, b = layer()
    y = mx.act_linear(z, w, b, "silu")
    g = torch.ones_like(y)
    got = torch.autograd.grad(y, (z, w, b), g)
    want = torch.autograd.grad(torch.nn.functional.linear(torch.nn.functional.silu(z), w, b), (z, w, b), g)
    for a, c in zip(got, want):
        torch.testing.assert_close(a, c, rtol=0.05, atol=0.05)  # z in 8 bits, a few roundings to bfloat16


def test_second_order_is_refused(mx):
    """A gradient penalty: its second-order terms must not be dropped without a word."""
    z, w, b = layer()
    y = mx.act_linear(z, w, b, "silu")
    (dz,) = torch.autograd.grad(y.float().square().sum(), z, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (dz.float().square().sum() + y.float().sum()).backward()


def test_backward_frees_the_checkpoint(mx):
    z, w, b = layer()
    loss = mx.act_linear(z, w, b, "silu").float().square().sum()
    (kept,) = mx.kept
    assert kept() is not None
    loss.backward()
    assert kept() is None and loss.isfinite()


def test_saved_tensor_hooks_see_the_checkpoint(mx):
    z, w, b = layer()
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.append(t.dtype), t.clone())[1], lambda t: t):
        y = mx.act_linear(z, w, b, "silu")
    assert torch.uint8 in seen and mx.kept[0]() is None  # what the hook made stands in for it
    got = torch.autograd.grad(y, (z, w, b), torch.ones_like(y))
    y = mx.act_linear(z, w, b, "silu")
    for a, c in zip(got, torch.autograd.grad(y, (z, w, b), torch.ones_like(y))):
        assert torch.equal(a, c)


def test_what_the_backward_pass_cannot_take_is_refused_in_the_forward(mx):
    z, w, b = layer(torch.float32)
    with pytest.raises(RuntimeError, match="z had dtype float32, expected one of float16, bfloat16"):
        mx.act_linear(z, w, b)
    h = lambda t: t.detach().half()
    for args in ((h(z), w, None), (h(z), h(w), b), (h(z), h(w).bfloat16(), None)):
        with pytest.raises(RuntimeError, match="the dtype of z"):
            mx.act_linear(*args)
    assert not mx.kept
