"""Cases for the microscaled low-precision operators (vorotracing_b200.mx).

Four operators, each in its plain form (elementary torch operations in 32 bits)
and through the package's entry points:

  act      h = act(z) with z kept in 8 bits for the backward pass, then
           dz = dh * act'(z8): one elementwise training step
  linear   the gradients of y = act(z) W^T + b from the 8-bit z:
           dz = (dy W) * act'(z8), dW = dy^T act(z8), db = sum dy
  linear4  y = act(q4(x) w4^T + b): product of two 4-bit microscaled matrices
  quant4   values of a matrix rounded to 4-bit microscaled blocks

Formats.  A row is cut into blocks of 32 columns (the last one may be short and
is padded with zeros).  8 bits: one exponent byte E a block, 2^(E - 127) the
power of two at or below the block's largest magnitude (E at least 7), values
code * 2^(E - 133) with codes in [-127, 127], rounded to nearest even.  4 bits:
E as for 8 bits but two less (at least 1), values e2m1 * 2^(E - 127) with e2m1
in {0, .5, 1, 1.5, 2, 3, 4, 6} and their negatives, rounded to nearest even and
saturated; code 8 is the sign, the low nibble is the even column.
"""
import math

import torch

own = False

BLOCK = 32
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ACTS = ("identity", "relu", "silu", "gelu_tanh")


def listed():
    return [
        # the hidden activations of a small colour decoder over one 1296x840 view
        {"name": "act_view", "op": "act", "rows": 1088640, "cols": 64, "dtype": "float16", "act": "silu"},
        # a small odd batch, where the launch is most of the time
        {"name": "act_odd", "op": "act", "rows": 1001, "cols": 193, "dtype": "float32", "act": "gelu_tanh"},
        # the decoder's colour head, training on one 1552x1040 view
        {"name": "linear_head", "op": "linear", "rows": 1614080, "cols": 64, "outs": 3, "dtype": "bfloat16", "act": "relu"},
        # a hidden layer of a wider decoder on one 1296x840 view
        {"name": "linear_hidden", "op": "linear", "rows": 1088640, "cols": 256, "outs": 256, "dtype": "bfloat16", "act": "silu"},
        # a patch of rays: latency
        {"name": "linear_patch", "op": "linear", "rows": 1000, "cols": 64, "outs": 64, "dtype": "bfloat16", "act": "silu"},
        # a wide layer: the matrix products bound it
        {"name": "linear_wide", "op": "linear", "rows": 8192, "cols": 4096, "outs": 4096, "dtype": "float16", "act": "gelu_tanh"},
        # one token through a wide layer: reading the weights
        {"name": "linear4_one", "op": "linear4", "rows": 1, "cols": 4096, "outs": 4096, "dtype": "bfloat16", "act": "identity"},
        # a ragged batch of few tokens
        {"name": "linear4_odd", "op": "linear4", "rows": 77, "cols": 1000, "outs": 333, "dtype": "float16", "act": "gelu_tanh"},
        # a decoder's first layer at inference on 192 = 3 * 8 * 8 texel values a ray
        {"name": "linear4_view", "op": "linear4", "rows": 1088640, "cols": 192, "outs": 64, "dtype": "bfloat16", "act": "silu"},
        # a large product: the tensor cores bound it
        {"name": "linear4_wide", "op": "linear4", "rows": 4096, "cols": 8192, "outs": 8192, "dtype": "bfloat16", "act": "identity"},
        # the texel map of a scene of a million cells (R = 8)
        {"name": "quant4_texels", "op": "quant4", "rows": 1000000, "cols": 192, "dtype": "float32"},
        # a small odd matrix
        {"name": "quant4_odd", "op": "quant4", "rows": 100, "cols": 75, "dtype": "bfloat16"},
    ]


def _spread(rng, lo, hi):
    """A whole number, uniform over the logarithm of the range."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("act", "linear", "linear", "linear4", "linear4", "quant4"))
    if op in ("act", "quant4"):
        cols = _spread(rng, 1, 8192)
        c = {"op": op, "rows": _spread(rng, 1, min(1 << 21, 60_000_000 // cols)), "cols": cols,
             "dtype": rng.choice(tuple(DTYPES))}
        return dict(c, act=rng.choice(ACTS)) if op == "act" else c
    cols, outs = _spread(rng, 8, 8192), _spread(rng, 1, 8192)
    if rng.random() < 0.5:  # half of the widths are ones that models have
        cols, outs = max(16, cols // 16 * 16), max(16, outs // 16 * 16)
    most = min(1 << 20, 100_000_000_000 // (cols * outs), 250_000_000 // max(cols, outs))
    return {"op": op, "rows": _spread(rng, 1, max(1, most)), "cols": cols, "outs": outs,
            "dtype": rng.choice(("bfloat16", "float16")), "act": rng.choice(ACTS)}


# ---------------------------------------------------------------- inputs

def _padded(cols):
    return -(-cols // BLOCK) * BLOCK


def _split(x):
    """(rows, blocks, 32) in 32 bits, zeros behind the last column."""
    rows, cols = x.shape
    y = torch.zeros((rows, _padded(cols)), dtype=torch.float32, device=x.device)
    y[:, :cols] = x
    return y.view(rows, -1, BLOCK)


def _exponent(blocks, least, lower):
    """Exponent byte of each block: that of the power of two at or below its largest magnitude, less `lower`."""
    top = blocks.abs().amax(dim=2)
    bits = (top.contiguous().view(torch.int32) >> 23) & 0xFF
    return torch.where(bits == 255, bits, torch.clamp(bits - lower, min=least))


def _pow2(e):
    """2^e for whole e in [-126, 127], exactly."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _codes8(x):
    """8-bit codes (rows, padded cols) and exponent bytes (rows, blocks)."""
    b = _split(x)
    e = _exponent(b, 7, 0)
    q = torch.round(b * _pow2(133 - e.clamp(max=254)).unsqueeze(2)).clamp(-127, 127)
    q = torch.where((e == 255).unsqueeze(2), torch.zeros_like(q), q)
    return q.to(torch.int8).view(x.shape[0], -1), e.to(torch.uint8)


def _values8(codes, exps, cols):
    rows = codes.shape[0]
    e = exps.to(torch.int32)
    s = torch.where(e == 255, torch.full_like(e, math.nan, dtype=torch.float32), _pow2(e.clamp(max=254) - 133))
    return (codes.view(rows, -1, BLOCK).float() * s.unsqueeze(2)).view(rows, -1)[:, :cols]


def _round4(b, e):
    """Blocks in units of 2^(e - 127), rounded to the nearest e2m1: index 0..7 of the magnitude."""
    v = (b * _pow2(127 - e.clamp(max=253)).unsqueeze(2)).abs()
    i = (v > 0.25).to(torch.uint8)
    for t, even in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        i += (v >= t) if even else (v > t)
    return i


def _codes4(x):
    """Packed 4-bit codes (rows, padded cols / 2) and exponent bytes (rows, blocks)."""
    b = _split(x)
    e = _exponent(b, 1, 2)
    i = _round4(b, e) + torch.signbit(b).to(torch.uint8) * 8
    i = torch.where((e == 255).unsqueeze(2), torch.zeros_like(i), i).view(x.shape[0], -1)
    return i[:, 0::2] | (i[:, 1::2] << 4), e.to(torch.uint8)


def _values4(codes, exps, cols):
    rows = codes.shape[0]
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    i = torch.stack((codes & 15, codes >> 4), dim=2).view(rows, -1, BLOCK)
    e = exps.to(torch.int32)
    s = torch.where(e == 255, torch.full_like(e, math.nan, dtype=torch.float32), _pow2(e.clamp(max=254) - 127))
    return (table[i.int()] * s.unsqueeze(2)).view(rows, -1)[:, :cols]


def _activations(rows, cols, gen, dtype):
    """Pre-activations: each column has a scale of its own, a few of them large, as hidden layers have."""
    col = torch.exp(0.5 * torch.randn(cols, generator=gen, device="cuda"))
    col[torch.rand(cols, generator=gen, device="cuda") < 0.02] *= 8
    out = torch.empty((rows, cols), dtype=dtype, device="cuda")
    step = max(1, (1 << 26) // cols)
    for at in range(0, rows, step):
        n = min(step, rows - at)
        out[at:at + n] = torch.randn((n, cols), generator=gen, device="cuda") * col
    return out


def _gradients(rows, cols, gen, dtype):
    """Upstream gradients: each ray's loss has a size of its own, and rays behind a mask have none.
    They get smaller with the batch, as under a loss scale that follows it."""
    row = torch.exp(torch.randn((rows, 1), generator=gen, device="cuda")) / math.sqrt(rows)
    row[torch.rand((rows, 1), generator=gen, device="cuda") < 0.1] = 0
    out = torch.empty((rows, cols), dtype=dtype, device="cuda")
    step = max(1, (1 << 26) // cols)
    for at in range(0, rows, step):
        n = min(step, rows - at)
        out[at:at + n] = torch.randn((n, cols), generator=gen, device="cuda") * row[at:at + n]
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, cols, dtype = case["rows"], case["cols"], DTYPES[case["dtype"]]
    s = dict(case, type=dtype)
    if case["op"] == "quant4":
        s["x"] = _activations(rows, cols, gen, dtype)
    elif case["op"] == "act":
        s["z"] = _activations(rows, cols, gen, dtype)
        s["dh"] = _gradients(rows, cols, gen, dtype)
    else:
        w = torch.randn((case["outs"], cols), generator=gen, device="cuda") / math.sqrt(cols)
        if case["op"] == "linear":
            # what the forward pass has left: 8-bit codes and exponents, made in parts
            s["codes"] = torch.empty((rows, _padded(cols)), dtype=torch.int8, device="cuda")
            s["exps"] = torch.empty((rows, _padded(cols) // BLOCK), dtype=torch.uint8, device="cuda")
            step = max(1, (1 << 26) // cols)
            z = _activations(rows, cols, gen, dtype)
            for at in range(0, rows, step):
                s["codes"][at:at + step], s["exps"][at:at + step] = _codes8(z[at:at + step])
            s["dy"] = _gradients(rows, case["outs"], gen, dtype)
            s["w"] = w.to(dtype)
        else:
            s["x"] = _activations(rows, cols, gen, dtype)
            s["wcodes"], s["wexps"] = _codes4(w)
            s["bias"] = torch.randn(case["outs"], generator=gen, device="cuda").to(dtype)
    return s


# ---------------------------------------------------------------- one pass

def _act(z, name):
    if name == "relu":
        return z * (z > 0)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu_tanh":
        return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).float()
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if name == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        p = 1 / (1 + torch.exp(-c * (z + 0.044715 * z * z * z)))
        return p * (1 + z * (1 - p) * c * (1 + 3 * 0.044715 * z * z))
    return torch.ones_like(z)


def _run_own(s):
    from vorotracing_b200 import mx

    if s["op"] == "act":
        h, ckpt = mx.act_checkpoint(s["z"], s["act"])
        return {"h": h, "dz": mx.act_backward(s["dh"], ckpt)}
    if s["op"] == "linear":
        ckpt = mx.Checkpoint(s["codes"], s["exps"], s["cols"], s["act"])
        dz, dw, db = mx.linear_backward(s["dy"], s["w"], ckpt, bias=True)
        return {"dz": dz, "dw": dw, "db": db}
    if s["op"] == "linear4":
        w = mx.MX4(s["wcodes"], s["wexps"], s["cols"])
        return {"y": mx.linear4(s["x"], w, bias=s["bias"], act=s["act"])}
    return {"x4": mx.quantize4(s["x"]).dequantize(s["type"])}


def _run_plain(s):
    t = s["type"]
    if s["op"] == "act":
        z = s["z"].float()
        z8 = _values8(*_codes8(z), s["cols"])
        return {"h": _act(z, s["act"]).to(t), "dz": (s["dh"].float() * _act_slope(z8, s["act"])).to(t)}
    if s["op"] == "linear":
        z8, dy = _values8(s["codes"], s["exps"], s["cols"]), s["dy"].float()
        dz = (dy @ s["w"].float()) * _act_slope(z8, s["act"])
        return {"dz": dz.to(t), "dw": (dy.t() @ _act(z8, s["act"])).to(t), "db": dy.sum(dim=0).to(t)}
    if s["op"] == "linear4":
        x4 = _values4(*_codes4(s["x"]), s["cols"])
        y = x4 @ _values4(s["wcodes"], s["wexps"], s["cols"]).t() + s["bias"].float()
        return {"y": _act(y, s["act"]).to(t)}
    return {"x4": _values4(*_codes4(s["x"]), s["cols"]).to(t)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    rows, cols = case["rows"], case["cols"]
    size = 4 if case["dtype"] == "float32" else 2
    n, kept = rows * cols, rows * _padded(cols) // BLOCK
    if case["op"] == "quant4":
        return {"bytes": 2 * n * size, "flops": 4 * n}
    if case["op"] == "act":  # z, dh in; h, dz out; the 8-bit form written and read
        return {"bytes": 4 * n * size + 2 * kept * (BLOCK + 1), "flops": 20 * n}
    outs = case["outs"]
    if case["op"] == "linear":  # 8-bit z, dy, w in; dz, dw, db out
        return {"bytes": kept * (BLOCK + 1) + size * (n + rows * outs + 2 * outs * cols + outs),
                "flops": 4 * n * outs + 10 * n + rows * outs}
    weights = outs * _padded(cols) // BLOCK * (BLOCK // 2 + 1)
    return {"bytes": weights + size * (n + rows * outs + outs), "flops": 2 * n * outs}


# ---------------------------------------------------------------- the definition, in 64 bits

def _logistic(x):
    return torch.special.expit(x)


def _act64(z, name):
    """(value, slope) of the activation, in 64 bits."""
    if name == "identity":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.clamp(z, min=0), (z > 0).double()
    if name == "silu":
        p = _logistic(z)
        return z * p, p + z * p * _logistic(-z)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 0.134145 * z ** 2)


def _block64(x, bits):
    """The values that a 64-bit matrix has after rounding to blocks of `bits` bits."""
    rows, cols = x.shape
    y = torch.nn.functional.pad(x.double(), (0, _padded(cols) - cols)).view(rows, -1, BLOCK)
    _, top = torch.frexp(y.abs().amax(dim=2, keepdim=True))
    top = top.double() - 1  # the largest magnitude is in [2^top, 2^(top + 1))
    if bits == 8:
        unit = torch.exp2(torch.clamp(top, min=-120) - 6)
        v = torch.clamp(torch.round(y / unit), -127, 127) * unit
    else:
        unit = torch.exp2(torch.clamp(top - 2, min=-126))
        m = torch.clamp(y.abs() / unit, max=6)
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(m, min=1))), max=2) - 1)
        v = torch.round(m / step) * step * unit * torch.sign(y)
    return v.view(rows, -1)[:, :cols]


def _from8(codes, exps, cols):
    unit = torch.exp2(exps.double() - 133).repeat_interleave(BLOCK, dim=1)
    return (codes.double() * unit)[:, :cols]


def _from4(codes, exps, cols):
    i = torch.stack((codes & 15, codes >> 4), dim=2).flatten(1).long()
    m = i & 7
    # e2m1: two exponent bits and one fraction bit; exponent 0 holds 0 and a half
    v = torch.where(m < 2, m.double() / 2, (1 + (m & 1).double() / 2) * torch.exp2((m >> 1).double() - 1))
    unit = torch.exp2(exps.double() - 127).repeat_interleave(BLOCK, dim=1)
    return (torch.where(i >= 8, -v, v) * unit)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    rows, cols = case["rows"], case["cols"]
    step = max(1, (1 << 26) // max(cols, case.get("outs", 1)))
    parts = [slice(at, min(at + step, rows)) for at in range(0, rows, step)]
    if case["op"] == "quant4":
        return {"x4": torch.cat([_block64(s["x"][p], 4) for p in parts])}
    if case["op"] == "act":
        h = torch.cat([_act64(s["z"][p].double(), case["act"])[0] for p in parts])
        dz = torch.cat([s["dh"][p].double() * _act64(_block64(s["z"][p], 8), case["act"])[1] for p in parts])
        return {"h": h, "dz": dz}
    if case["op"] == "linear":
        dz, dw, db = [], 0, 0
        w = s["w"].double()
        for p in parts:
            dy = s["dy"][p].double()
            h, slope = _act64(_from8(s["codes"][p], s["exps"][p], cols), case["act"])
            dz.append(dy @ w * slope)
            dw, db = dw + dy.t() @ h, db + dy.sum(dim=0)
        return {"dz": torch.cat(dz), "dw": dw, "db": db}
    w = _from4(s["wcodes"], s["wexps"], cols).t()
    y = [_act64(_block64(s["x"][p], 4) @ w + s["bias"].double(), case["act"])[0] for p in parts]
    return {"y": torch.cat(y)}
