"""The ray decoder on a rendered view: trained through 8-bit checkpoints, run in 4 bits."""
import numpy as np
import pytest
import torch

import mx_reference as R

pytestmark = pytest.mark.gpu


def view(h=48, w=64):
    from vorotracing_b200 import scene as sc
    from vorotracing_b200.render import InferScene

    s = sc.make_scene(2048, 11, False, 8, cache=False)
    rays = sc.pinhole_rays(sc.intrinsics(w, h), sc.look_at((0.0, 0.0, 3.0), up=(0, 1, 0)), w, h)
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    scene = InferScene(d(s["points"]), d(s["density"]), d(s["adj"]), d(s["offs"]), d(s["diffuse"]), d(s["specular"]))
    rays = d(rays)
    return scene.render(rays, weight_threshold=0.01), rays


def test_decoder_trains_on_a_view_and_runs_in_4_bits():
    from vorotracing_b200 import mx
    from vorotracing_b200.decoder import RayDecoder, ray_features

    rgba, rays = view()
    x = ray_features(rgba, rays)
    assert x.shape == (48, 64, 16) and x.dtype == torch.bfloat16
    target = torch.sin(3 * rgba[..., :3].float()) * (1 + rays[..., 3:6].float()) * 0.5  # a tone curve that depends on the view
    torch.manual_seed(0)
    decoder = RayDecoder(features=16, hidden=64, layers=2)
    opt = torch.optim.Adam(decoder.parameters(), lr=5e-3)
    losses = []
    for _ in range(60):
        loss = (decoder(x).float() - target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < 0.2 * losses[0]
    y, y4 = decoder(x).detach().float(), decoder.quantized()(x).float()
    # one layer in 4 bits is off by about a tenth of its output; three in a row stay well below the target's own spread
    assert (y - y4).square().mean() < 0.25 * (target - target.mean((0, 1))).square().mean()
    mx.raise_errors()


def test_decoder_gradients_are_those_of_the_8_bit_layers():
    """Against the layers written out in 64 bits at the 8-bit values of each layer's own input."""
    from vorotracing_b200 import mx
    from vorotracing_b200.decoder import RayDecoder

    torch.manual_seed(1)
    decoder = RayDecoder(features=16, hidden=32, layers=1, outs=3)
    x = torch.randn(200, 16, device="cuda").bfloat16().requires_grad_()
    g = torch.randn(200, 3, device="cuda").bfloat16()
    decoder(x).backward(g)
    w0, w1 = (w.detach() for w in decoder.weights)
    z0 = torch.nn.functional.linear(x.detach(), w0, decoder.biases[0].detach())
    _, ckpt = mx.act_checkpoint(z0, "silu")
    dz, dw1, db1 = mx.linear_backward(g, w1, ckpt)
    z8 = ckpt.dequantize().double()
    assert torch.equal(decoder.weights[1].grad, dw1) and torch.equal(decoder.biases[1].grad, db1)
    want = (g.double() @ w1.double()) * R.slope(z8, "silu")
    u = R.UNIT[torch.bfloat16]
    R.assert_within(dz, want, 2 * u * want.abs() + 2.0 ** -16 * (g.double().abs() @ w1.double().abs()), "dz")
    _, ckpt0 = mx.act_checkpoint(x.detach(), "identity")
    dx, dw0, db0 = mx.linear_backward(dz, w0, ckpt0)
    assert torch.equal(x.grad, dx) and torch.equal(decoder.weights[0].grad, dw0) and torch.equal(decoder.biases[0].grad, db0)


def test_decoder_refuses():
    from vorotracing_b200.decoder import RayDecoder

    with pytest.raises(ValueError, match="at least 1"):
        RayDecoder(16, layers=0)
    with pytest.raises(RuntimeError, match="unknown activation"):
        RayDecoder(16, act="sine")
