"""Microscaled 4-bit formats in numpy float64, straight from their definition (test oracle)."""
import numpy as np

BLOCK = {"MXFP4": 32, "NVFP4": 16}
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)])[:127]
NAN_BYTE = {"MXFP4": 0xFF, "NVFP4": 0x7F}
STEPS = {"MXFP4": (0, 1, -1), "NVFP4": (0, 1, -1, 2, -2, 3, 4, 5)}


def nearest(v, grid):
    """Index of the entry of an ascending grid nearest to v >= 0, ties to the even index."""
    i = np.clip(np.searchsorted(grid, v), 1, len(grid) - 1)
    lo, hi = v - grid[i - 1], grid[i] - v
    return np.where((lo < hi) | ((lo == hi) & ((i - 1) % 2 == 0)), i - 1, i)


def scale_value(byte, fmt):
    byte = np.asarray(byte, np.int64)
    if fmt == "MXFP4":
        return np.where(byte == 255, np.nan, np.ldexp(1.0, np.minimum(byte, 254).astype(int) - 127))
    return np.where(byte == 127, np.nan, E4M3[np.minimum(byte, 126)])


def first_scale(a, fmt):
    """Scale byte of a block from its largest magnitude (already divided by the tensor scale)."""
    if fmt == "MXFP4":
        return np.where(a > 0, np.clip(np.frexp(a)[1] - 1 - 2 + 127, 0, 254), 0)
    return nearest(np.minimum(a / 6.0, 448.0), E4M3)


def block_codes(x, s):
    """Codes (sign in bit 3) of x [..., b] against steps s [...]."""
    s = s[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(s > 0, np.abs(x) / s, 0.0)
    c = nearest(np.minimum(q, 6.0), LEVELS)
    return c + 8 * np.signbit(x)


def quantize(x, fmt, g=1.0, qw=None):
    """x [rows, n] -> (codes [rows, nb, block] 0..15, scale bytes [rows, nb]); n padded with zeros."""
    b = BLOCK[fmt]
    rows, n = x.shape
    p = -(-n // b) * b
    xb = np.pad(np.asarray(x, np.float64), ((0, 0), (0, p - n))).reshape(rows, p // b, b) / g
    bad = ~np.isfinite(xb).all(2)
    xb = np.where(bad[..., None], 0.0, xb)
    byte = first_scale(np.abs(xb).max(2), fmt)
    codes = block_codes(xb, scale_value(byte, fmt))
    if qw is not None:
        w = np.pad(np.asarray(qw, np.float64), (0, p - n)).reshape(1, p // b, b)
        first, best, err = byte, byte, None
        for k in STEPS[fmt]:
            cb = np.where(first > 0, np.clip(first + k, 0, 254 if fmt == "MXFP4" else 126), first)
            s = scale_value(cb, fmt)
            cc = block_codes(xb, s)
            e = (w * (np.abs(xb) - LEVELS[cc & 7] * s[..., None]) ** 2).sum(2)
            if err is None:
                best, codes, err = cb, cc, e
            else:
                better = e < err
                best, codes = np.where(better, cb, best), np.where(better[..., None], cc, codes)
                err = np.where(better, e, err)
        byte = best
    return np.where(bad[..., None], 0, codes), np.where(bad, NAN_BYTE[fmt], byte)


def values(codes, byte, fmt, g=1.0, n=None):
    v = np.where(codes >= 8, -1.0, 1.0) * LEVELS[codes & 7] * scale_value(byte, fmt)[..., None] * g
    v = v.reshape(v.shape[0], -1)
    return v if n is None else v[:, :n]


def unpack(codes, scales, fmt, rows, n):
    """An operand's arrays (numpy uint8) -> (codes [rows, nb, block], bytes [rows, nb]), nb of the padded row."""
    q = np.stack([codes & 15, codes >> 4], 2).reshape(rows, -1)
    t = scales.transpose(0, 3, 2, 1, 4)
    t = t.reshape(t.shape[0] * 128, -1)[:rows]
    return q.reshape(rows, -1, BLOCK[fmt]).astype(np.int64), t.astype(np.int64)


def pack(codes, byte, fmt, n):
    """(codes [rows, nb, block], bytes [rows, nb]) -> an operand's arrays."""
    b, rows = BLOCK[fmt], codes.shape[0]
    p = -(-n // 256) * 256
    q = np.zeros((rows, p), np.uint8)
    q[:, :codes.shape[1] * b] = codes.reshape(rows, -1)
    rp = -(-rows // 128) * 128
    s = np.zeros((rp, p // b), np.uint8)
    s[:rows, :byte.shape[1]] = byte
    t = s.reshape(rp // 128, 4, 32, p // b // 4, 4).transpose(0, 3, 2, 1, 4)
    return q[:, 0::2] | (q[:, 1::2] << 4), np.ascontiguousarray(t)


def container(codes, byte):
    """MXFP4 blocks as GGUF holds them: [rows, nb * 17]."""
    c = codes.astype(np.uint8)
    raw = np.concatenate([byte[..., None].astype(np.uint8), c[..., :16] | (c[..., 16:] << 4)], 2)
    return raw.reshape(raw.shape[0], -1)
