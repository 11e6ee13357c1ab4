"""Cases for the microscaled 4-bit operators (perm_b200.mx4, and MXFP4 in perm_b200.kquant):
quantisation and its inverse, the product of two 4-bit operands, the product of activations
with frozen 4-bit weights, and that product's gradient.

A 4-bit operand is what a user's program keeps between calls:
  codes   uint8 [rows, P/2], P = n rounded up to 256, element 2j of a row in the low four bits
          of byte j (e2m1: sign, two exponent bits, one mantissa bit); padding is zero
  scales  uint8, one byte per block of 32 (MXFP4, e8m0) or 16 (NVFP4, e4m3), in tiles of 128
          rows x 4 blocks: [rows/128, blocks/4, 32, 4, 4], byte (r, j, k) of a tile belonging to
          row 32 j + r and block k; rows padded to 128, blocks to the padded row; padding zero
  scale   a power of two that multiplies the whole tensor (NVFP4; 1 for MXFP4)
"""
import torch

own = False

BLOCK = {"MXFP4": 32, "NVFP4": 16}
DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
# tensor scales of NVFP4 operands: activations of a few units, weights of about 0.02
GX, GW = 2.0 ** -5, 2.0 ** -14


# ------------------------------------------------------------------------------- cases

def listed():
    return [
        # one token's hidden state on its way into a 4-bit product (latency)
        dict(name="quantize_token", kind="quantize", fmt="MXFP4", dtype="bf16", rows=1, n=4096),
        # a prefill batch's hidden states
        dict(name="quantize_prefill", kind="quantize", fmt="NVFP4", dtype="bf16", rows=8192, n=4096),
        # encoding one ffn matrix of an 8B model into the GGUF container with its imatrix
        dict(name="encode_ffn_imatrix", kind="encode", fmt="MXFP4", dtype="f32", rows=14336, n=4096),
        # a weight of odd shape, importance-weighted, into the operand layout
        dict(name="quantize_weight_odd", kind="quantize_weight", fmt="NVFP4", dtype="f32", rows=1025, n=2000),
        # one token through a small projection, both operands in 4 bits (latency)
        dict(name="matmul_token", kind="matmul", fmt="MXFP4", dtype="bf16", rows=1, n=1024, out=2048),
        # a ragged batch, float32 result
        dict(name="matmul_ragged", kind="matmul", fmt="MXFP4", dtype="f32", rows=333, n=2050, out=1500),
        # prefill through the ffn of an 8B model, both operands in 4 bits
        dict(name="matmul_prefill", kind="matmul", fmt="NVFP4", dtype="bf16", rows=8192, n=4096, out=14336),
        # decoding one token: the ffn's weights stream once
        dict(name="linear_token", kind="linear", fmt="MXFP4", dtype="bf16", rows=1, n=4096, out=14336),
        # a small decode batch through the down projection
        dict(name="linear_batch", kind="linear", fmt="NVFP4", dtype="f16", rows=12, n=14336, out=4096),
        # prefill with activations kept in bfloat16
        dict(name="linear_prefill", kind="linear", fmt="MXFP4", dtype="bf16", rows=4096, n=4096, out=14336),
        # distillation through frozen weights: forward and the gradient of the input
        dict(name="train_step", kind="train", fmt="MXFP4", dtype="bf16", rows=4096, n=4096, out=4096),
        # the same in float32 at a small odd shape
        dict(name="train_odd_f32", kind="train", fmt="NVFP4", dtype="f32", rows=97, n=1000, out=515),
    ]


def _log(rng, lo, hi):
    """A whole number of lo .. hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["quantize", "encode", "quantize_weight", "matmul", "linear", "linear", "train"])
    fmt = rng.choice(["MXFP4", "NVFP4"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "encode":
        return dict(kind=kind, fmt="MXFP4", dtype="f32", rows=_log(rng, 1, 14336), n=32 * _log(rng, 1, 128))
    if kind == "quantize_weight":
        return dict(kind=kind, fmt=fmt, dtype="f32", rows=_log(rng, 1, 8192), n=_log(rng, 16, 4096))
    if kind == "quantize":
        return dict(kind=kind, fmt=fmt, dtype=dtype, rows=_log(rng, 1, 8192), n=_log(rng, 16, 4096))
    rows = _log(rng, 1, 4096)
    n, out = _log(rng, 64, 8192), _log(rng, 64, 8192)
    if rng.random() < 0.4:
        n, out = n // 64 * 64, out // 64 * 64
    return dict(kind=kind, fmt=fmt, dtype=dtype, rows=rows, n=n, out=out)


# ------------------------------------------------------------------------------- plain forms

def _pad(x, cols):
    return torch.nn.functional.pad(x, (0, cols - x.shape[1]))


def _padded(n):
    return -(-n // 256) * 256


def _tile(s):
    """[rows, blocks] scale bytes -> the operand's tiles."""
    rows, nb = s.shape
    r = -(-rows // 128) * 128
    s = torch.nn.functional.pad(s, (0, 0, 0, r - rows))
    return s.view(r // 128, 4, 32, nb // 4, 4).permute(0, 3, 2, 1, 4).contiguous()


def _untile(t, rows):
    a, c = t.shape[:2]
    return t.permute(0, 3, 2, 1, 4).reshape(a * 128, c * 4)[:rows]


def _e4m3_round(v):
    """Nearest e4m3 code (0 .. 126) of values >= 0 in 64 bits, ties to even, saturating."""
    e = torch.frexp(v)[1].clamp(min=-5) - 1                     # v = m 2^e, 1 <= m < 2 (or below)
    k = torch.round(torch.ldexp(v, 3 - e))                      # eighths: 8 .. 16 (0 .. 8 below 2^-6)
    return ((e + 6) * 8 + k).clamp(max=126.0).to(torch.int32)   # a carry into 16 goes to the next exponent


def _e4m3_value(c):
    c = c.to(torch.int32)
    e, m = c >> 3, (c & 7).double()
    return torch.where(e == 0, torch.ldexp(m, torch.full_like(e, -9)), torch.ldexp(8 + m, e - 10))


def _scale_value(c, fmt):
    """What a scale byte stands for, in 64 bits."""
    if fmt == "MXFP4":
        return torch.ldexp(torch.ones_like(c, dtype=torch.float64), c.to(torch.int32) - 127)
    return _e4m3_value(c)


def _first_scale(amax, fmt, g):
    """The scale byte of a block from its largest magnitude (64 bits)."""
    if fmt == "MXFP4":
        c = (torch.frexp(amax)[1] - 3 + 127).clamp(0, 254)
        return torch.where(amax > 0, c, torch.zeros_like(c)).to(torch.int32)
    return _e4m3_round(amax / (6 * g))


def _code(x, s):
    """Magnitude code 0 .. 7 of x against the step s: comparisons with the borders, ties to even."""
    a = x.abs()
    c = ((a > 0.25 * s).to(torch.uint8) + (a >= 0.75 * s) + (a > 1.25 * s) + (a >= 1.75 * s)
         + (a > 2.5 * s) + (a >= 3.5 * s) + (a > 5 * s))
    return torch.where(s > 0, c, torch.zeros_like(c))


def _grid(dtype, dev):
    return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=dtype, device=dev)


def _quantize(x, fmt, g, qw=None):
    """x [rows, n] -> (codes uint8 [rows, n/2], scale bytes [rows, blocks]), n a multiple of 256."""
    rows, n = x.shape
    b = BLOCK[fmt]
    xb = x.double().view(rows, n // b, b)
    c = _first_scale(xb.abs().amax(2), fmt, g)
    if qw is None:
        m = _code(xb, (_scale_value(c, fmt) * g).unsqueeze(2))
    else:
        step = torch.tensor([0, 1, -1] if fmt == "MXFP4" else [0, 1, -1, 2, -2, 3, 4, 5], device=x.device)
        top = 254 if fmt == "MXFP4" else 126
        cand = torch.where((c > 0).unsqueeze(0), (c.unsqueeze(0) + step.view(-1, 1, 1)).clamp(0, top), c.unsqueeze(0))
        s = (_scale_value(cand, fmt) * g).unsqueeze(3)
        mag = _code(xb.unsqueeze(0), s)
        d = xb.abs().unsqueeze(0) - _grid(torch.float64, x.device)[mag.long()] * s
        err = (qw.double().view(1, 1, n // b, b) * (d * d)).sum(3)
        pick = err.argmin(0, keepdim=True)
        c = cand.gather(0, pick)[0]
        m = mag.gather(0, pick.unsqueeze(3).expand(1, rows, n // b, b))[0]
    q = (m + 8 * torch.signbit(xb).to(torch.uint8)).view(rows, n)
    return q[:, 0::2] | (q[:, 1::2] << 4), c.to(torch.uint8)


def _values(codes, scales, fmt, g, n, dtype=torch.float32):
    """The values [rows, n] of packed codes and scale bytes."""
    q = torch.stack((codes & 15, codes >> 4), 2).view(codes.shape[0], -1)
    v = _grid(torch.float64, codes.device)[q.long()].view(codes.shape[0], -1, BLOCK[fmt])
    return (v * (_scale_value(scales, fmt) * g).unsqueeze(2)).view(codes.shape[0], -1)[:, :n].to(dtype)


def _operand_values(w):
    return _values(w["codes"], _untile(w["scales"], w["rows"]), w["fmt"], w["scale"], w["n"])


# ------------------------------------------------------------------------------- states

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(case, g):
    """N(0, 1) with log-normal channel scales, as hidden states have."""
    x = torch.randn(case["rows"], case["n"], generator=g, device="cuda")
    return (x * torch.exp(0.7 * torch.randn(case["n"], generator=g, device="cuda"))).to(DTYPE[case["dtype"]])


def _weights(rows, n, g):
    return torch.randn(rows, n, generator=g, device="cuda") * 0.02


def _operand(rows, n, fmt, g):
    """A weight matrix of `rows` outputs in 4 bits."""
    scale = 1.0 if fmt == "MXFP4" else GW
    codes, sb = _quantize(_pad(_weights(rows, n, g), _padded(n)), fmt, scale)
    return dict(codes=codes, scales=_tile(sb), fmt=fmt, rows=rows, n=n, scale=scale)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(kind=case["kind"], fmt=case["fmt"], dtype=DTYPE[case["dtype"]])
    if case["kind"] in ("encode", "quantize_weight"):
        s["x"] = _weights(case["rows"], case["n"], g)
        # mean squares of the inputs, as an imatrix holds them
        s["qw"] = torch.exp(1.4 * torch.randn(case["n"], generator=g, device="cuda"))
        s["scale"] = 1.0 if case["fmt"] == "MXFP4" else GW
        return s
    s["x"] = _activations(case, g)
    s["scale"] = 1.0 if case["fmt"] == "MXFP4" else GX
    if case["kind"] != "quantize":
        s["w"] = _operand(case["out"], case["n"], case["fmt"], g)
    if case["kind"] == "train":
        s["x"].requires_grad_(True)
        s["dy"] = torch.randn(case["rows"], case["out"], generator=g, device="cuda").to(DTYPE[case["dtype"]])
    return s


# ------------------------------------------------------------------------------- one pass

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_plain(s):
    x, fmt = s["x"], s["fmt"]
    n = x.shape[1]
    if s["kind"] in ("encode", "quantize_weight"):
        qw = torch.nn.functional.pad(s["qw"], (0, _padded(n) - n))
        return _values(*_quantize(_pad(x, _padded(n)), fmt, s["scale"], qw), fmt, s["scale"], n)
    if s["kind"] == "quantize":
        return _values(*_quantize(_pad(x, _padded(n)), fmt, s["scale"]), fmt, s["scale"], n).to(s["dtype"])
    w = _operand_values(s["w"])
    if s["kind"] == "matmul":
        a = _values(*_quantize(_pad(x, _padded(n)), fmt, s["scale"]), fmt, s["scale"], n)
        return (a @ w.t()).to(s["dtype"])
    y = (x.detach().float() @ w.t()).to(s["dtype"])
    if s["kind"] == "linear":
        return y
    return {"y": y, "dx": (s["dy"].float() @ w).to(s["dtype"])}


def _run_own(s):
    from perm_b200 import kquant, mx4
    x = s["x"]
    if s["kind"] == "encode":
        return kquant.DEQUANTIZE[s["fmt"]](kquant.QUANTIZE[s["fmt"]](x, s["qw"]), x.shape[1])
    if s["kind"] in ("quantize", "quantize_weight"):
        return mx4.dequantize(mx4.quantize(x, s["fmt"], qw=s.get("qw"), tensor_scale=s["scale"]), s["dtype"])
    h = s["w"]
    w = mx4.Mx4Tensor(h["codes"], h["scales"], h["fmt"], h["rows"], h["n"], h["scale"])
    if s["kind"] == "matmul":
        return mx4.matmul(mx4.quantize(x, s["fmt"], tensor_scale=s["scale"]), w, s["dtype"])
    y = mx4.linear(x, w)
    if s["kind"] == "linear":
        return y
    return {"y": y.detach(), "dx": torch.autograd.grad(y, x, s["dy"])[0]}


# ------------------------------------------------------------------------------- floors

def work(case):
    rows, n, size = case["rows"], case["n"], SIZE[case["dtype"]]
    packed = 0.5 + 1 / BLOCK[case["fmt"]]
    if case["kind"] in ("quantize", "encode", "quantize_weight"):
        # read, write the packed form, read it, write its values; a compare and a product for each value
        weighted = {"MXFP4": 3, "NVFP4": 8}[case["fmt"]] if case["kind"] != "quantize" else 0
        return {"bytes": rows * n * (2 * size + 2 * packed), "flops": rows * n * (3 + 5 * weighted)}
    out = case["out"]
    one = rows * n * size + out * n * packed + rows * out * size
    if case["kind"] == "matmul":
        one += 2 * rows * n * packed
    times = 2 if case["kind"] == "train" else 1
    return {"bytes": times * one, "flops": times * 2 * rows * n * out}


# ------------------------------------------------------------------------------- 64 bits

_LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _nearest(v):
    """Nearest e2m1 level of |v| by distance; of two equally near, the one with the even place."""
    a = v.abs()
    best, level = torch.full_like(a, float("inf")), torch.zeros_like(a)
    for i in (0, 2, 4, 6, 1, 3, 5, 7):                # even places first: they keep a tie
        d = (a - _LEVELS[i]).abs()
        nearer = d < best
        best, level = torch.where(nearer, d, best), torch.where(nearer, torch.full_like(a, _LEVELS[i]), level)
    return torch.copysign(level, v)


def _e4m3_table():
    t = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    return torch.tensor(t[:127], dtype=torch.float64, device="cuda")


def _exact_values(x, fmt, g, qw=None):
    """Quantised values of x, block by block, straight from the definition."""
    rows, n = x.shape
    b = BLOCK[fmt]
    p = -(-n // b) * b
    xb = torch.nn.functional.pad(x.double(), (0, p - n)).view(rows, p // b, b)
    top = xb.abs().amax(2)
    if fmt == "MXFP4":
        first = torch.floor(torch.log2(top.clamp(min=2.0 ** -140))) - 2
        first = torch.where(torch.exp2(first + 3) <= top, first + 1, first)      # log2 may round across a power
        first = torch.where(torch.exp2(first + 2) > top, first - 1, first).clamp(-127, 127)
        steps = [torch.exp2((first + k).clamp(-127, 127)) for k in ((0,) if qw is None else (0, 1, -1))]
    else:
        t = _e4m3_table()
        v = (top / (6 * g)).clamp(max=448.0)
        hi = torch.searchsorted(t, v.contiguous()).clamp(max=126)
        lo = (hi - 1).clamp(min=0)
        dl, dh = v - t[lo], t[hi] - v
        at = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
        offs = (0,) if qw is None else (0, 1, -1, 2, -2, 3, 4, 5)
        steps = [g * t[torch.where(at > 0, (at + k).clamp(0, 126), at)] for k in offs]
    got = err = None
    for s in steps:
        s = s.unsqueeze(2)
        q = torch.where(s > 0, _nearest(xb / torch.where(s > 0, s, torch.ones_like(s))) * s, torch.zeros_like(xb))
        if qw is None:
            got = q
            break
        e = (torch.nn.functional.pad(qw.double(), (0, p - n)).view(1, p // b, b) * (xb - q) ** 2).sum(2, keepdim=True)
        better = torch.ones_like(e, dtype=torch.bool) if got is None else e < err
        got = q if got is None else torch.where(better, q, got)
        err = e if err is None else torch.where(better, e, err)
    return got.reshape(rows, p)[:, :n]


def _exact_weights(w):
    """The 64-bit values of an operand, element by element."""
    rows, n, b = w["rows"], w["n"], BLOCK[w["fmt"]]
    r = torch.arange(rows, device="cuda").view(-1, 1)
    k = torch.arange(n, device="cuda").view(1, -1)
    nib = (w["codes"][:, : (n + 1) // 2].repeat_interleave(2, 1)[:, :n].to(torch.int32) >> (4 * (k % 2))) & 15
    blk = torch.arange(-(-n // b), device="cuda").view(1, -1)
    byte = w["scales"][r // 128, blk // 4, r % 32, (r % 128) // 32, blk % 4]
    if w["fmt"] == "MXFP4":
        s = torch.exp2(byte.double() - 127)
    else:
        s = _e4m3_table()[byte.long()]
    level = torch.tensor(_LEVELS, dtype=torch.float64, device="cuda")[(nib & 7).long()]
    v = torch.where(nib >= 8, -level, level)
    return v * s.repeat_interleave(b, 1)[:, :n] * w["scale"]


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach()
    if case["kind"] in ("encode", "quantize_weight", "quantize"):
        return _exact_values(x, s["fmt"], s["scale"], s.get("qw"))
    w = _exact_weights(s["w"])
    if case["kind"] == "matmul":
        return torch.matmul(_exact_values(x, s["fmt"], s["scale"]), w.t())
    y = torch.matmul(x.double(), w.t())
    if case["kind"] == "linear":
        return y
    return {"y": y, "dx": torch.matmul(s["dy"].double(), w)}
