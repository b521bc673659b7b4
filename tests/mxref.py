"""MXFP4 and the block norm restated with numpy in 64 bits (test infrastructure)."""
import numpy as np

NUMBERS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def bf16_bits(x):
    """f32 -> bf16 bits, nearest even (NaN stays NaN)"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + np.uint32(0x7FFF) + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def bf16_values(bits):
    return (np.asarray(bits).astype(np.uint32) << 16).view(np.float32)


def quantize(x):
    """f32 rows (R, K) -> codes (R, K) uint8, scale bytes (R, K / 32) uint8"""
    r, k = x.shape
    b = x.astype(np.float64).reshape(r, k // 32, 32)
    top = np.abs(b).max(-1)
    bad = ~np.isfinite(b).all(-1)
    _, e = np.frexp(np.where(bad | (top == 0), 1.0, top))          # top = m 2^e, m in [0.5, 1)
    e = np.where(top == 0, -127, np.maximum(e - 1 - 2, -127))
    a = np.abs(np.where(bad[..., None], 0.0, b)) / np.ldexp(1.0, e)[..., None]
    d = np.abs(a[..., None] - NUMBERS)
    near = d.min(-1, keepdims=True)
    # nearest; of two equally near numbers the even code
    is_near = d == near
    first = is_near.argmax(-1)
    last = 7 - is_near[..., ::-1].argmax(-1)
    code = np.where(first % 2 == 0, first, last) + 8 * np.signbit(b)
    code = np.where(bad[..., None], 0, code)
    return code.reshape(r, k).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, byte):
    """64-bit values of codes (R, K), scale bytes (R, K / 32)"""
    r, k = codes.shape
    v = np.where(codes & 8, -1.0, 1.0) * NUMBERS[codes & 7]
    s = np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(np.int64) - 127))
    return (v.reshape(r, k // 32, 32) * s[..., None]).reshape(r, k)


def planes(codes, byte):
    """the MXFP4_SPLIT bytes"""
    return np.concatenate([(codes[:, 0::2] | codes[:, 1::2] << 4).reshape(-1), byte.reshape(-1)]).astype(np.uint8)


def unplanes(buf, rows, k):
    q = buf[:rows * k // 2].reshape(rows, k // 2)
    c = np.empty((rows, k), np.uint8)
    c[:, 0::2], c[:, 1::2] = q & 15, q >> 4
    return c, buf[rows * k // 2:rows * k // 2 + rows * (k // 32)].reshape(rows, k // 32)


def blocks(codes, byte):
    """the MXFP4 blocks (R, K / 32, 17)"""
    r, k = codes.shape
    c = codes.reshape(r, k // 32, 32)
    return np.concatenate([byte[..., None], c[..., :16] | c[..., 16:] << 4], -1).astype(np.uint8)


def norm(v, kind, eps):
    """kind: 0 none, 1 layer, 2 RMS"""
    if kind == 0:
        return v
    if kind == 1:
        v = v - v.mean(-1, keepdims=True)
    return v / np.sqrt((v * v).mean(-1, keepdims=True) + eps)
