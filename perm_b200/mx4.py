"""Microscaled 4-bit operands: quantisation, products with them, and the products' gradient.

    from perm_b200 import mx4
    w = mx4.quantize(W, "MXFP4", qw)           # frozen weights [out, n], importance-weighted scales
    y = mx4.linear(x, w)                       # x bf16 / f16 / f32 [..., n] -> [..., out]; x gets a gradient
    a = mx4.quantize(x, "MXFP4")               # activations in 4 bits
    y = mx4.matmul(a, w, torch.bfloat16)       # both operands in 4 bits

Values are e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign) times a block scale: "MXFP4" has blocks of
32 with an e8m0 scale (a power of two), "NVFP4" blocks of 16 with an e4m3 scale and one tensor
scale.  A block of MXFP4 takes the exponent floor(log2 max) - 2, one of NVFP4 the e4m3 nearest to
max / 6 / tensor_scale; values round to nearest even and saturate at 6.  With column weights qw
(as kquant's imatrix path has them) each block tries several scales and keeps the one with the
least sum of qw (x - value)^2, formed in 64 bits.  A NaN or an infinity makes its block NaN.

The GGUF container of MXFP4 is in kquant (QUANTIZE["MXFP4"], DEQUANTIZE["MXFP4"]); from_gguf
turns its bytes into an operand.

Calls only enqueue work on the current stream of the tensors' device, and every tensor of a call
is on that device.  Products accumulate in float32 and round once.  Their kernels bound every
wait; status() raises if one ran out.
"""
import copy
import math

import torch
from torch.autograd import forward_ad as _forward

from . import _native as nat

BLOCK = {"MXFP4": 32, "NVFP4": 16}
_ID = nat.MX4_ID
_DTYPE = {torch.bfloat16: nat.CP_MX4_BF16, torch.float16: nat.CP_MX4_F16, torch.float32: nat.CP_MX4_F32}
# A call on one token takes a few microseconds on the device, so the host's part is kept short: the
# stream's address comes from torch directly (a Stream object costs more than the rest of the checks).
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_MIN_SCALE, _MAX_SCALE = 2.0 ** -126, (2.0 - 2.0 ** -23) * 2.0 ** 127   # float32's normal numbers
_workspace = {}   # sizes of a linear call -> workspace bytes


class Mx4Tensor:
    """A 4-bit operand [rows, n].

    codes   uint8 [rows, P/2], P = n rounded up to 256: element 2j of a row in the low half of
            byte j, zero past n
    scales  uint8, tiles of 128 rows x 4 blocks, [ceil(rows/128), P/(4 block), 32, 4, 4]: entry
            [i, g, r, j, k] is the scale of row 128 i + 32 j + r, block 4 g + k; zero past n and
            past the last row
    tensor_scale  a positive float that multiplies every value"""
    __slots__ = ("fmt", "rows", "n", "tensor_scale", "dev", "_codes", "_scales", "_buf", "_cp", "_sp")

    def __init__(self, codes, scales, fmt, rows, n, tensor_scale=1.0):
        if fmt not in BLOCK:
            raise ValueError(f"unknown 4-bit format {fmt!r}")
        pitch = (n + 255) // 256 * 128
        if rows < 0 or n <= 0 or codes.dtype != torch.uint8 or codes.shape != (rows, pitch) or not codes.is_contiguous():
            raise ValueError(f"codes must be a contiguous uint8 [{rows}, {pitch}]")
        if scales.dtype != torch.uint8 or not scales.is_contiguous() or \
                scales.numel() != (rows + 127) // 128 * 256 * pitch // BLOCK[fmt]:
            raise ValueError(f"scales must be contiguous uint8 tiles of {rows} rows and {pitch * 2 // BLOCK[fmt]} blocks")
        if codes.device != scales.device:
            raise ValueError("codes and scales must be on one device")
        if not _MIN_SCALE <= tensor_scale <= _MAX_SCALE:
            raise ValueError("tensor_scale must be positive and within float32's normal range")
        self.fmt, self.rows, self.n, self.tensor_scale = fmt, rows, n, tensor_scale
        self.dev = codes.get_device()   # CUDA device index, -1 on the host
        self._codes, self._scales, self._buf = codes, scales, None
        self._cp, self._sp = codes.data_ptr(), scales.data_ptr()

    @classmethod
    def _new(cls, like, fmt, rows, n, tensor_scale, buf=None):
        """An operand on like's device, not yet filled: one allocation (or `buf`, which is one), of which
        codes and scales are views made when they are asked for."""
        q = cls.__new__(cls)
        pitch = (n + 255) // 256 * 128
        at = (rows * pitch + 255) // 256 * 256
        q._buf = buf if buf is not None else like.new_empty((at + (rows + 127) // 128 * (256 // BLOCK[fmt]) * pitch,), dtype=torch.uint8)
        q.fmt, q.rows, q.n, q.tensor_scale, q.dev = fmt, rows, n, tensor_scale, like.get_device()
        q._codes = q._scales = None
        q._cp = q._buf.data_ptr()
        q._sp = q._cp + at
        return q

    @property
    def codes(self):
        if self._codes is None:
            pitch = (self.n + 255) // 256 * 128
            self._codes = self._buf[:self.rows * pitch].view(self.rows, pitch)
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            pitch = (self.n + 255) // 256 * 128
            self._scales = self._buf[(self.rows * pitch + 255) // 256 * 256:].view(-1, pitch // (2 * BLOCK[self.fmt]), 32, 4, 4)
        return self._scales

    @property
    def shape(self):
        return (self.rows, self.n)

    @property
    def device(self):
        return (self._codes if self._buf is None else self._buf).device

    # Copies are made through __init__, so that the addresses are those of their own tensors.
    def _rest(self):
        return self.fmt, self.rows, self.n, self.tensor_scale

    def __copy__(self):
        return Mx4Tensor(self.codes, self.scales, *self._rest())

    def __deepcopy__(self, memo):
        return Mx4Tensor(copy.deepcopy(self.codes, memo), copy.deepcopy(self.scales, memo), *self._rest())

    def __reduce__(self):   # clones: a view is written with all that shares its storage
        return Mx4Tensor, (self.codes.clone(), self.scales.clone(), *self._rest())

    def _tensors(self):
        return (self._codes, self._scales) if self._buf is None else (self._buf,)

    def _over(self, tensors):
        """This operand over tensors in the place of its own (all of _tensors())."""
        if len(tensors) == 2:
            return Mx4Tensor(*tensors, *self._rest())
        return Mx4Tensor._new(tensors[0], *self._rest(), buf=tensors[0])

    def __repr__(self):
        return f"Mx4Tensor({self.fmt}, [{self.rows}, {self.n}], tensor_scale={self.tensor_scale}, device={self.device})"


def _refuse_host(what):
    raise nat.CudaPathError(f"{what}: tensors must be on a CUDA device")


def _call(idx, fn, what, *args):
    """fn(*args, stream) on device idx's current stream, with idx the current device."""
    if idx == _current_device():
        rc = fn(*args, _raw_stream(idx))
    else:
        with torch.cuda.device(idx):
            rc = fn(*args, _raw_stream(idx))
    if rc:
        nat.check(rc, what)


def tensor_scale_for(x):
    """A power of two g for quantize(x, "NVFP4", tensor_scale=g): the least with
    max |x| / (6 g) <= 448, so the largest block scale uses e4m3's range.  Reads x on the host."""
    m = float(x.detach().abs().amax()) if x.numel() else 0.0
    if not math.isfinite(m):
        raise ValueError("tensor_scale_for: x has values that are not finite")
    if m == 0.0:
        return 1.0
    f, e = math.frexp(m / (6.0 * 448.0))
    return math.ldexp(1.0, max(-99, min(99, e - 1 if f == 0.5 else e)))


def quantize(x, fmt, qw=None, tensor_scale=1.0):
    """x [rows, n] (bf16, f16 or f32; any row stride) -> Mx4Tensor.  qw: non-negative column
    weights [n], or None.  tensor_scale: a power of two (1 for MXFP4).  x gets no gradient."""
    if fmt not in BLOCK:
        raise ValueError(f"unknown 4-bit format {fmt!r}")
    if not x.is_cuda:
        _refuse_host("mx4.quantize")
    dt = _DTYPE.get(x.dtype)
    if dt is None or x.dim() != 2 or x.shape[1] == 0:
        raise ValueError("mx4.quantize expects a bf16, f16 or f32 matrix [rows, n], n > 0")
    rows, n = x.shape
    if not x.is_contiguous() and (x.stride(1) != 1 or x.stride(0) < n):
        x = x.contiguous()
    if qw is not None:
        if qw.shape != (n,) or qw.device != x.device:
            raise ValueError(f"qw must hold {n} column weights on x's device")
        qw = qw.to(torch.float32).contiguous()
    q = Mx4Tensor._new(x, fmt, rows, n, tensor_scale)
    _call(q.dev, nat.lib().cp_mx4_quantize, "mx4.quantize", _ID[fmt], dt, x.data_ptr(), rows, n, x.stride(0),
          None if qw is None else qw.data_ptr(), tensor_scale, q._cp, q._sp)
    return q


def dequantize(q, dtype=torch.float32):
    """The values of an operand, [rows, n] in `dtype` (bf16, f16 or f32)."""
    dt = _DTYPE.get(dtype)
    if dt is None:
        raise ValueError("mx4.dequantize: dtype must be bf16, f16 or f32")
    if q.dev < 0:
        _refuse_host("mx4.dequantize")
    out = (q._buf if q._codes is None else q._codes).new_empty((q.rows, q.n), dtype=dtype)
    _call(q.dev, nat.lib().cp_mx4_dequantize, "mx4.dequantize", _ID[q.fmt], q._cp, q._sp, q.rows, q.n, q.tensor_scale, dt, out.data_ptr())
    return out


def from_gguf(raw, n):
    """GGUF MXFP4 bytes (uint8 CUDA [rows, n/32 * 17], as kquant.QUANTIZE["MXFP4"] gives) -> Mx4Tensor."""
    if not raw.is_cuda:
        _refuse_host("mx4.from_gguf")
    if n <= 0 or n % 32:
        raise ValueError(f"cannot reshape a row of {n} values into 32-value blocks")
    if raw.dtype != torch.uint8 or raw.dim() != 2 or raw.shape[1] != n // 32 * 17:
        raise ValueError(f"raw must be uint8 [rows, {n // 32 * 17}]")
    raw = raw.contiguous()
    q = Mx4Tensor._new(raw, "MXFP4", raw.shape[0], n, 1.0)
    _call(q.dev, nat.lib().cp_mx4_from_gguf, "mx4.from_gguf", raw.data_ptr(), q.rows, n, q._cp, q._sp)
    return q


def matmul(a, w, dtype=torch.bfloat16):
    """a w^T for two operands of one format: a [T, n], w [out, n] -> [T, out] in `dtype` (no gradient)."""
    dt = _DTYPE.get(dtype)
    if dt is None:
        raise ValueError("mx4.matmul: dtype must be bf16, f16 or f32")
    if a.fmt != w.fmt or a.n != w.n:
        raise ValueError(f"mx4.matmul: {a!r} and {w!r} must have one format and one n")
    if a.dev != w.dev:
        raise ValueError("mx4.matmul: operands must be on one device")
    scale = a.tensor_scale * w.tensor_scale
    if not _MIN_SCALE <= scale <= _MAX_SCALE:
        raise ValueError("mx4.matmul: the product of the tensor scales must be within float32's normal range")
    if a.dev < 0:
        _refuse_host("mx4.matmul")
    y = (w._buf if w._codes is None else w._codes).new_empty((a.rows, w.rows), dtype=dtype)
    _call(a.dev, nat.lib().cp_mx4_matmul, "mx4.matmul", _ID[w.fmt], a._cp, a._sp, a.rows, w._cp, w._sp, w.rows, w.n,
          scale, dt, y.data_ptr())
    return y


def _product(x, w, transpose, what):
    """x [..., K] times w^T (transpose: times w)."""
    dt = _DTYPE.get(x.dtype)
    K, out = (w.rows, w.n) if transpose else (w.n, w.rows)
    shape = x.shape
    if dt is None:
        raise ValueError(f"{what} expects bf16, f16 or f32, not {x.dtype}")
    if not shape or shape[-1] != K:
        raise ValueError(f"{what}: the last dimension must be {K}, not {tuple(shape)}")
    dev = w.dev
    if x.get_device() != dev:
        raise ValueError(f"{what}: the operands must be on one device")
    if dev < 0:
        _refuse_host(what)
    if len(shape) == 2:
        T = shape[0]
        y = x.new_empty((T, out))
    else:
        T = math.prod(shape[:-1])
        y = x.new_empty((*shape[:-1], out))
        x = x.reshape(T, K)
    ld = K
    if not x.is_contiguous():
        if x.stride(1) != 1 or T > 1 and x.stride(0) < K:
            x = x.contiguous()
        else:
            ld = x.stride(0)
    L, p = nat.lib(), x.data_ptr()
    key = (dev, dt, T, ld, w.rows, w.n, transpose, p & 15)
    need = _workspace.get(key)
    if need is None:
        if len(_workspace) > 4096:
            _workspace.clear()
        need = _workspace[key] = L.cp_mx4_linear_workspace_bytes(dt, p, T, ld, w.rows, w.n, transpose)
    ws = x.new_empty((need,), dtype=torch.uint8) if need else None
    _call(dev, L.cp_mx4_linear, what, _ID[w.fmt], dt, p, T, ld, w._cp, w._sp, w.rows, w.n, w.tensor_scale, transpose,
          y.data_ptr(), ws.data_ptr() if need else None, need)
    return y


class _Product(torch.autograd.Function):
    """The product and its transpose are each other's gradient (the weights are frozen)."""

    @staticmethod
    def forward(ctx, x, w, transpose):
        ctx.w, ctx.transpose = w, transpose
        own = w._buf if w._codes is None else w._codes
        if not own.is_inference():   # those have no version and cannot be saved
            ctx.save_for_backward(*w._tensors())
        return _product(x, w, transpose, "mx4.linear_grad" if transpose else "mx4.linear")

    @staticmethod
    def backward(ctx, dy):
        w, saved = ctx.w, ctx.saved_tensors   # raises if the weights were written since
        if saved and saved[0] is not (w._codes if w._buf is None else w._buf):
            w = w._over(saved)
        if torch.is_grad_enabled() or _forward._current_level >= 0:   # create_graph, or dy has a tangent: a gradient itself
            return _Product.apply(dy, w, 1 - ctx.transpose), None, None
        return _product(dy, w, 1 - ctx.transpose, "mx4.linear (backward)"), None, None

    @staticmethod
    def jvp(ctx, tangent, *_):
        return _Product.apply(tangent, ctx.w, ctx.transpose)


def linear(x, w):
    """x w^T: x [..., n] (bf16, f16 or f32), w [out, n] -> [..., out] in x's type.  x is taken as it is; only
    float32 values of up to 16 rows may be off by a unit in the last place (2^-23), and values below 2^-110
    are taken as multiples of 2^-133.  NVFP4's sums are formed
    before the tensor scale: |x| up to 2^100 keeps them finite.  x gets a gradient (reverse and forward mode,
    also of second order; torch.func and vmap raise); the weights are frozen."""
    if x.requires_grad and torch.is_grad_enabled() or _forward._current_level >= 0:
        return _Product.apply(x, w, 0)
    return _product(x, w, 0, "mx4.linear")


def linear_grad(dy, w):
    """The gradient of linear(x, w) with respect to x: dy w, dy [..., out] -> [..., n]."""
    if dy.requires_grad and torch.is_grad_enabled() or _forward._current_level >= 0:
        return _Product.apply(dy, w, 1)
    return _product(dy, w, 1, "mx4.linear_grad")


def status(device=None):
    """Raise CudaPathError if a bounded wait in an earlier product on `device` ran out (its result
    is incomplete); synchronises the current stream."""
    nat.torch_cuda()
    idx = None if device is None else torch.device(device).index
    if idx is None:   # a device without a number is the current one
        idx = torch.cuda.current_device()
    _call(idx, nat.lib().cp_mx4_status, "mx4.status")


class Linear(torch.nn.Module):
    """torch.nn.Linear with frozen 4-bit weights (hessians.collect_hessians hooks it like one, so
    the Hessians of later layers can be collected from an encoded model's own activations)."""

    def __init__(self, weight, bias=None):
        super().__init__()
        self.out_features, self.in_features = weight.shape
        self.fmt, self.tensor_scale = weight.fmt, weight.tensor_scale
        # buffers of their own: a view would save and move with everything it shares its storage with
        self.register_buffer("codes", weight.codes.clone())
        self.register_buffer("scales", weight.scales.clone())
        self.bias = None if bias is None else torch.nn.Parameter(bias.detach().clone())

    @classmethod
    def from_linear(cls, linear, fmt="MXFP4", qw=None, tensor_scale=None):
        """Encodes a torch.nn.Linear on a CUDA device (NVFP4's tensor scale from its weights unless given)."""
        w = linear.weight.detach()
        if tensor_scale is None:
            tensor_scale = tensor_scale_for(w) if fmt == "NVFP4" else 1.0
        return cls(quantize(w, fmt, qw, tensor_scale), linear.bias)

    @property
    def weight4(self):
        return Mx4Tensor(self.codes, self.scales, self.fmt, self.out_features, self.in_features, self.tensor_scale)

    def get_extra_state(self):
        """What a saved state holds beside codes, scales and bias: the format's id and the tensor scale."""
        return torch.tensor([_ID[self.fmt], self.tensor_scale], dtype=torch.float64)

    def set_extra_state(self, state):
        fmt, scale = state.tolist()
        if fmt != _ID[self.fmt]:
            raise ValueError(f"the saved weights are not {self.fmt}")
        self.tensor_scale = scale

    def forward(self, x):
        y = linear(x, self.weight4)
        return y if self.bias is None else y + self.bias.to(y.dtype)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, fmt={self.fmt}, bias={self.bias is not None}"
