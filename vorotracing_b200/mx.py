"""Microscaled low-precision operators for a learned layer beside the tracer.

No counterpart in the reference.  Two formats, both in blocks of 32 columns
with one power-of-two scale a block (``include/vorotracing_b200.h`` has the
layouts): 8 bits for what a training step keeps of a layer's pre-activations,
4 bits for weights and activations at inference.

    h, ckpt = act_checkpoint(z, "silu")        # h = act(z); z kept in 8 bits
    y = h @ weight.t() + bias
    dz, dw, db = linear_backward(dy, weight, ckpt)   # from the 8-bit z

    w4 = quantize4(weight)                     # once
    y = linear4(x, w4, bias, "silu")           # act(q4(x) w4^T + b)

``act_linear`` is the training pair as an autograd function, and alone records
gradients.  Tensors live on a CUDA device, kernels run on torch's current
stream, outputs are new tensors there; matrices may have any row stride.
Elementwise operators take float32, float16 and bfloat16, products the 16-bit
types.  A block of 32 columns that holds a NaN or an infinity is NaN in either
format.

Every wait inside a product's kernel ends after about a second.  A kernel that
gave up has outputs that are not valid: the next product called after it has
ended raises, as an asynchronous error of CUDA does, and ``raise_errors`` waits
for the device and tells at once.  A loop of training steps learns of it in the
step after; what must not use such outputs calls ``raise_errors`` first.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import check, lib

BLOCK = 32
ACTS = {"identity": 0, "relu": 1, "silu": 2, "gelu_tanh": 3}
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_P, _U64, _U32, _I = C.c_void_p, C.c_uint64, C.c_uint32, C.c_int

_ARGS = {
    "vt_mx8_checkpoint": (_P, _I, _U64, _U32, _U64, _I, _P, _P, _P, _P),
    "vt_mx8_act_bwd": (_P, _I, _U64, _U32, _U64, _P, _P, _I, _P, _P),
    "vt_mx8_dequantize": (_P, _P, _U64, _U32, _I, _P, _P),
    "vt_mx8_linear_bwd_workspace_bytes": (_U64, _U32, _U32, _I),
    "vt_mx8_linear_bwd": (_P, _U64, _P, _U64, _I, _U64, _U32, _U32, _P, _P, _I, _P, _P, _P, _P,
                          _U64, _P, _P),
    "vt_mx4_quantize": (_P, _I, _U64, _U32, _U64, _P, _P, _P),
    "vt_mx4_dequantize": (_P, _P, _U64, _U32, _I, _P, _P),
    "vt_mx4_linear_workspace_bytes": (_U64, _U32, _U32, _I),
    "vt_mx4_linear": (_P, _U64, _I, _U64, _U32, _U32, _P, _P, _P, _I, _P, _P, _U64, _P, _P),
    "vt_wait_check": (_P, _P),
    "vt_error_word_create": (_P,),
}
_fn = {}
_get_device = torch.cuda.current_device
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_error_words = {}


def _error_word(index: int) -> int:
    """Address of the word where a product's kernel on that device reports that one of its waits has run out: host
    memory, which is not a graph's even if the first product is captured."""
    word = _error_words.get(index)
    if word is None:
        p = _P()
        check(_call("vt_error_word_create")(C.addressof(p)), "vt_error_word_create")
        word = _error_words.setdefault(index, C.c_uint32.from_address(p.value))
    if word.value:
        _gave_up(word)
    return C.addressof(word)


def _gave_up(word):
    code, word.value = word.value, 0
    _fail(f"a microscaled product's kernel gave up waiting (status {code}); its outputs "
          "are not valid")


def raise_errors(device=None):
    """Waits for the device and raises if a product's kernel gave up there since the last call."""
    i = torch.cuda.current_device() if device is None else torch.device(device).index
    if i is None:
        i = torch.cuda.current_device()
    word = _error_words.get(i)
    if word is not None:
        torch.cuda.synchronize(i)
        if word.value:
            _gave_up(word)


def _call(name):
    """The C entry point with its argument types declared, so that plain integers can be passed."""
    f = _fn.get(name)
    if f is None:
        f = getattr(lib(), name)
        f.argtypes = _ARGS[name]
        f.restype = C.c_uint64 if name.endswith("_bytes") else C.c_int
        _fn[name] = f
    return f


def _fail(msg: str):
    raise RuntimeError(msg)


def _act_code(act: str) -> int:
    code = ACTS.get(act)
    if code is None:
        _fail(f"unknown activation {act!r}, expected one of {', '.join(ACTS)}")
    return code


def _matrix(t, name: str, types=_DTYPES):
    """A tensor as rows of its last dimension with unit column stride: (tensor, rows, cols, row
    stride, type code)."""
    code = types.get(t.dtype)
    if code is None or not t.is_cuda:
        if not t.is_cuda:
            _fail(f"{name} must be on CUDA device")
        _fail(f"{name} had dtype {str(t.dtype).replace('torch.', '')}, expected one of "
              + ", ".join(str(d).replace("torch.", "") for d in types))
    shape = t.shape
    if len(shape) == 2:
        rows, cols = shape
        stride, unit = t.stride()
        if (unit == 1 or cols <= 1) and (stride >= cols or rows <= 1):
            return t, rows, cols, stride if rows > 1 else cols, code
    elif not shape:
        _fail(f"{name} must have at least one dimension")
    t = t.contiguous()
    rows, cols = 1, shape[-1]
    for n in shape[:-1]:
        rows *= n
    return t, rows, cols, cols, code


_PRODUCT_TYPES = {torch.float16: 1, torch.bfloat16: 2}


def _launch(name: str, index: int, *args):
    """Calls an entry point on the tensors' device and torch's current stream there."""
    f = _fn.get(name) or _call(name)
    if index < 0:  # as what was loaded to the host is
        _fail("the operand must be on CUDA device")
    if index == _get_device():
        status = f(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = f(*args, _raw_stream(index))
    if status:
        check(status, name)


def _unaligned(ptr: int, stride: int) -> bool:
    """Whether 16-bit rows at that address and stride do not all start on 16 bytes."""
    return bool(ptr % 16 or stride % 8)


class _Blocks:
    """Codes and exponent bytes of a matrix, as two tensors or as one buffer that holds both.

    Only tensors and sizes are kept, and addresses are taken from the tensors at each call, so that an
    object's copies, and what is loaded of it elsewhere, have memory of their own."""

    __slots__ = ("cols", "rows", "_codes", "_exps", "_buf")
    _dtype: torch.dtype
    _per_block: int
    _align: int

    def _take(self, codes, exps, cols: int):
        what, per, blocks = type(self).__name__, self._per_block, -(-cols // BLOCK)
        if codes.dtype is not self._dtype or exps.dtype is not torch.uint8:
            _fail(f"{what}: codes must be {str(self._dtype).replace('torch.', '')} and exponents uint8")
        shape = codes.shape
        if len(shape) != 2 or shape[1] != blocks * per or exps.shape != (shape[0], blocks):
            _fail(f"{what}: {cols} columns take codes (rows, {blocks * per}) and exponents "
                  f"(rows, {blocks}), got {tuple(shape)} and {tuple(exps.shape)}")
        if not codes.is_cuda or codes.get_device() != exps.get_device():
            _fail(f"{what}: codes and exponents must be on the same CUDA device")
        if not codes.is_contiguous() or not exps.is_contiguous():
            _fail(f"{what}: codes and exponents must be contiguous")
        if codes.data_ptr() % self._align:
            _fail(f"{what}: codes must be {self._align}-byte aligned")
        self._codes, self._exps, self._buf = codes, exps, None
        self.cols, self.rows = cols, shape[0]

    def _new(self, like, rows: int, cols: int):
        self.cols, self.rows, self._codes, self._exps = cols, rows, None, None
        self._buf = like.new_empty(rows * -(-cols // BLOCK) * (self._per_block + 1), dtype=torch.uint8)

    def _place(self):
        """(device index, address of the codes, address of the exponents)"""
        buf = self._buf
        if buf is not None:
            p = buf.data_ptr()
            return buf.get_device(), p, p + self.rows * -(-self.cols // BLOCK) * self._per_block
        return self._codes.get_device(), self._codes.data_ptr(), self._exps.data_ptr()

    @property
    def device_index(self) -> int:
        return (self._codes if self._buf is None else self._buf).get_device()

    @property
    def codes(self) -> torch.Tensor:
        if self._buf is None:
            return self._codes
        width = -(-self.cols // BLOCK) * self._per_block
        return self._buf[:self.rows * width].view(self._dtype).view(self.rows, width)

    @property
    def exps(self) -> torch.Tensor:
        if self._buf is None:
            return self._exps
        blocks = -(-self.cols // BLOCK)
        return self._buf[self.rows * blocks * self._per_block:].view(self.rows, blocks)

    def _dequantize(self, entry: str, dtype) -> torch.Tensor:
        code = _DTYPES.get(dtype)
        if code is None:
            _fail(f"cannot dequantise to {str(dtype).replace('torch.', '')}")
        index, codes, exps = self._place()
        out = (self._codes if self._buf is None else self._buf).new_empty((self.rows, self.cols), dtype=dtype)
        _launch(entry, index, codes, exps, self.rows, self.cols, code, out.data_ptr())
        return out


class Checkpoint(_Blocks):
    """A matrix of pre-activations in 8 bits and the activation it goes through.

    codes (rows, 32 B) int8, exps (rows, B) uint8, B = ceil(cols / 32)."""

    __slots__ = ("act", "_act", "dtype")  # dtype: z's, None if unknown
    _dtype, _per_block, _align = torch.int8, BLOCK, 32

    def __init__(self, codes, exps, cols: int, act: str):
        self._act = _act_code(act)
        self.act, self.dtype = act, None
        self._take(codes, exps, cols)

    @classmethod
    def _of(cls, buf, rows: int, cols: int, act: str):
        """A checkpoint from its buffer."""
        ckpt = cls.__new__(cls)
        ckpt.act, ckpt._act, ckpt.dtype, ckpt._codes, ckpt._exps = act, _act_code(act), None, None, None
        ckpt._buf, ckpt.rows, ckpt.cols = buf, rows, cols
        return ckpt

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """The 8-bit values, (rows, cols)."""
        return self._dequantize("vt_mx8_dequantize", dtype)


class MX4(_Blocks):
    """A matrix in 4-bit microscaled blocks: codes (rows, 16 B) uint8, two columns a
    byte with the even one in the low nibble, exps (rows, B) uint8."""

    __slots__ = ()
    _dtype, _per_block, _align = torch.uint8, BLOCK // 2, 16

    def __init__(self, codes, exps, cols: int):
        self._take(codes, exps, cols)

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """The 4-bit values, (rows, cols)."""
        return self._dequantize("vt_mx4_dequantize", dtype)


def act_checkpoint(z: torch.Tensor, act: str = "silu"):
    """(act(z), 8-bit checkpoint of z) for z (..., cols), in one pass."""
    code = _act_code(act)
    m, rows, cols, stride, dtype = _matrix(z, "z")
    h = m.new_empty(z.shape)
    ckpt = Checkpoint.__new__(Checkpoint)
    ckpt.act, ckpt._act, ckpt.dtype = act, code, m.dtype
    ckpt._new(m, rows, cols)
    index, codes, exps = ckpt._place()
    _launch("vt_mx8_checkpoint", index, m.data_ptr(), dtype, rows, cols, stride, code, h.data_ptr(), codes, exps)
    return h, ckpt


def act_backward(dh: torch.Tensor, ckpt: Checkpoint) -> torch.Tensor:
    """dz = dh * act'(z8), in dh's type and shape."""
    m, rows, cols, stride, dtype = _matrix(dh, "dh")
    if rows != ckpt.rows or cols != ckpt.cols:
        _fail(f"dh had {rows} rows of {cols}, the checkpoint has {ckpt.rows} of {ckpt.cols}")
    index, codes, exps = ckpt._place()
    if m.get_device() != index:
        _fail("dh must be on the same device as the checkpoint")
    dz = m.new_empty(dh.shape)
    _launch("vt_mx8_act_bwd", index, m.data_ptr(), dtype, rows, cols, stride, codes, exps, ckpt._act, dz.data_ptr())
    return dz


def linear_backward(dy: torch.Tensor, weight: torch.Tensor, ckpt: Checkpoint, bias: bool = True,
                    need_dz: bool = True, need_dw: bool = True):
    """Gradients of y = act(z) W^T + b from the 8-bit checkpoint of z.

    dy (..., outs) and weight (outs, cols) in the same 16-bit type.  Returns
    (dz, dw, db) in that type: dz (..., cols) = (dy W) * act'(z8), dw (outs,
    cols) = dy^T act(z8) and db (outs) = column sums of dy; None for those not
    asked for.  act(z8) enters dw rounded to that type, as the forward pass's
    own activations do; a checkpoint of values beyond float16's range takes
    bfloat16 products."""
    m, rows, outs, dy_stride, dtype = _matrix(dy, "dy", _PRODUCT_TYPES)
    w, w_rows, cols, w_stride, w_type = _matrix(weight, "weight", _PRODUCT_TYPES)
    if w_rows != outs or weight.dim() != 2:
        _fail(f"weight had shape {tuple(weight.shape)}, expected ({outs}, columns)")
    if w_type != dtype:
        _fail("weight must have the dtype of dy")
    if dtype == 1 and ckpt.dtype not in (torch.float16, None):
        _fail("float16 products take a checkpoint of float16 values, which have its range; this one was made of "
              + str(ckpt.dtype).replace("torch.", ""))
    if rows != ckpt.rows or cols != ckpt.cols:
        _fail(f"dy has {rows} rows and weight {cols} columns, the checkpoint has {ckpt.rows} "
              f"rows of {ckpt.cols}")
    index, codes, exps = ckpt._place()
    if m.get_device() != index or w.get_device() != index:
        _fail("weight and the checkpoint must be on the same device as dy")
    dz = m.new_empty((*dy.shape[:-1], cols)) if need_dz else None
    dw = m.new_empty((outs, cols)) if need_dw else None
    db = m.new_empty(outs) if bias else None
    m_ptr, w_ptr = m.data_ptr(), w.data_ptr()
    n = _call("vt_mx8_linear_bwd_workspace_bytes")(
        rows, cols, outs, _unaligned(m_ptr, dy_stride) + 2 * _unaligned(w_ptr, w_stride))
    ws = m.new_empty(n, dtype=torch.uint8) if n else None
    _launch("vt_mx8_linear_bwd", index, m_ptr, dy_stride, w_ptr, w_stride, dtype, rows, cols, outs,
            codes, exps, ckpt._act, dz.data_ptr() if need_dz else None,
            dw.data_ptr() if need_dw else None, db.data_ptr() if bias else None,
            ws.data_ptr() if n else None, n, _error_word(index))
    return dz, dw, db


class _ActLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, weight, bias, act):
        h, ckpt = act_checkpoint(z, act)
        ctx.shape, ctx.has_bias = (ckpt.rows, ckpt.cols, act), bias is not None
        ctx.save_for_backward(weight, ckpt._buf)  # freed by the backward pass, seen by saved-tensor hooks
        return torch.nn.functional.linear(h, weight, bias)

    @staticmethod
    @torch.autograd.function.once_differentiable  # the kernels record no graph: second derivatives are refused
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        weight, buf = ctx.saved_tensors
        dz, dw, db = linear_backward(dy, weight, Checkpoint._of(buf, *ctx.shape),
                                     bias=ctx.has_bias and need[2], need_dz=need[0],
                                     need_dw=need[1])
        return dz, dw, db, None


def act_linear(z: torch.Tensor, weight: torch.Tensor, bias=None, act: str = "silu"):
    """y = act(z) W^T + b for training, the product by torch: between forward
    and backward only the 8-bit form of z is kept (33/32 byte a value), neither
    z nor act(z).  First derivatives only.

    z, weight and bias have one 16-bit type; under torch.autocast they may have
    any and are brought to its type, with gradients in their own."""
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        z, weight, bias = (t if t is None or t.dtype is torch.float64 else t.to(dtype) for t in (z, weight, bias))
        with torch.autocast("cuda", enabled=False):
            return act_linear(z, weight, bias, act)
    # what linear_backward would refuse is refused here, before anything is computed
    if z.dtype not in _PRODUCT_TYPES:
        _fail(f"z had dtype {str(z.dtype).replace('torch.', '')}, expected one of "
              + ", ".join(str(d).replace("torch.", "") for d in _PRODUCT_TYPES) + " (or torch.autocast)")
    if weight.dtype is not z.dtype or (bias is not None and bias.dtype is not z.dtype):
        _fail("weight and bias must have the dtype of z")
    return _ActLinear.apply(z, weight, bias, act)


def quantize4(x: torch.Tensor) -> MX4:
    """x (..., cols) in 4-bit microscaled blocks, as (rows, cols)."""
    m, rows, cols, stride, dtype = _matrix(x, "x")
    q = MX4.__new__(MX4)
    q._new(m, rows, cols)
    index, codes, exps = q._place()
    _launch("vt_mx4_quantize", index, m.data_ptr(), dtype, rows, cols, stride, codes, exps)
    return q


def linear4(x: torch.Tensor, w: MX4, bias=None, act: str = "identity") -> torch.Tensor:
    """y = act(q4(x) w4^T + bias): x (..., cols) in a 16-bit type is rounded to
    4 bits on the way, w is the weight (outs, cols) in 4 bits, bias (outs) has
    x's type.  y (..., outs) has x's type."""
    code = _act_code(act)
    m, rows, cols, stride, dtype = _matrix(x, "x", _PRODUCT_TYPES)
    outs = w.rows
    index, codes, exps = w._place()
    if cols != w.cols:
        _fail(f"x had {cols} columns, the weight has {w.cols}")
    if m.get_device() != index:
        _fail("the weight must be on the same device as x")
    b_ptr = None
    if bias is not None:
        if bias.dtype is not x.dtype or bias.shape != (outs,):
            _fail(f"bias must have the dtype of x and shape ({outs},)")
        if bias.get_device() != index:
            _fail("bias must be on the same device as x")
        bias = bias.contiguous()
        b_ptr = bias.data_ptr()
    y = m.new_empty((*x.shape[:-1], outs))
    m_ptr = m.data_ptr()
    n = _call("vt_mx4_linear_workspace_bytes")(rows, cols, outs, _unaligned(m_ptr, stride))
    ws = m.new_empty(n, dtype=torch.uint8) if n else None
    _launch("vt_mx4_linear", index, m_ptr, stride, dtype, rows, cols, outs, codes, exps, b_ptr, code,
            y.data_ptr(), ws.data_ptr() if n else None, n, _error_word(index))
    return y
