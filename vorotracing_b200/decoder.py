"""A small learned decoder on what the tracer renders.

``RayDecoder`` maps per-ray features (a traced colour and alpha, the view
direction, depths) to colours through a few linear layers; no counterpart in
the reference, whose colours come from the cells' texels alone.  With a ray a
row, activations outnumber weights by far, so they decide both of its forms:

  training   ``forward`` keeps each layer's pre-activations in 8 bits for the
             backward pass (``mx.act_linear``), half of what bfloat16 takes
  inference  ``quantized`` gives the same layers with weights in 4 bits
             (``mx.linear4``); each layer rounds its input to 4 bits on the way,
             which costs an image some 13 dB where it was not trained for it

    decoder = RayDecoder(features=16, hidden=64, layers=2)
    colours = decoder(ray_features(rgba, rays))     # trains as any module
    fast = decoder.quantized()
    colours = fast(ray_features(rgba, rays))
    mx.raise_errors()   # waits; raises if a kernel gave up (else the next call of a layer does)
"""
from __future__ import annotations

import torch

from . import mx


def ray_features(rgba: torch.Tensor, rays: torch.Tensor, extra=None, dtype=torch.bfloat16) -> torch.Tensor:
    """Features of each ray: traced rgba (..., 4), the first- and second-order terms of its
    unit direction (9) and any extra columns (..., E), padded to a multiple of 16 columns."""
    d = torch.nn.functional.normalize(rays[..., 3:6].float(), dim=-1)
    x, y, z = d.unbind(-1)
    parts = [rgba.float(), d, torch.stack((x * y, y * z, x * z, x * x - y * y, 3 * z * z - 1, torch.ones_like(x)), -1)]
    if extra is not None:
        parts.append(extra.float())
    f = torch.cat(parts, dim=-1)
    return torch.nn.functional.pad(f, (0, -f.size(-1) % 16)).to(dtype)


class RayDecoder(torch.nn.Module):
    """features -> hidden (x layers) -> outs, SiLU between the layers.

    Parameters in a 16-bit type train as they are, those in float32 under torch.autocast."""

    def __init__(self, features: int, hidden: int = 64, layers: int = 2, outs: int = 3, act: str = "silu",
                 device="cuda", dtype=torch.bfloat16):
        super().__init__()
        if layers < 1:
            raise ValueError("layers must be at least 1")
        mx._act_code(act)
        self.act = act
        widths = [features] + [hidden] * layers + [outs]
        self.weights = torch.nn.ParameterList(
            torch.nn.Parameter((torch.randn(o, i, device=device) / i ** 0.5).to(dtype)) for i, o in zip(widths, widths[1:]))
        self.biases = torch.nn.ParameterList(
            torch.nn.Parameter(torch.zeros(o, device=device, dtype=dtype)) for o in widths[1:])

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        z = mx.act_linear(x, self.weights[0], self.biases[0], "identity")
        for w, b in zip(self.weights[1:], self.biases[1:]):
            z = mx.act_linear(z, w, b, self.act)
        return z

    def quantized(self) -> "QuantizedRayDecoder":
        """The decoder with 4-bit weights, as they are now."""
        return QuantizedRayDecoder(self)


class QuantizedRayDecoder:
    def __init__(self, decoder: RayDecoder):
        self.act = decoder.act
        self.layers = [(mx.quantize4(w.detach()), b.detach().clone()) for w, b in zip(decoder.weights, decoder.biases)]

    @torch.no_grad()
    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        for w, b in self.layers[:-1]:
            x = mx.linear4(x, w, b.to(x.dtype), self.act)
        w, b = self.layers[-1]
        return mx.linear4(x, w, b.to(x.dtype))
