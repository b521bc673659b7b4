"""8-bit rows, rotary positions over several axes and cross attention restated with numpy in 64 bits (test infrastructure)."""
import numpy as np


def i8_quantize(x):
    """f32 rows (R, K) -> integers (R, K) int8, scales (R,) f32"""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(-1)
    z = np.where(bad[:, None], np.float32(0), x)
    d = np.maximum(np.abs(z).max(-1), np.float32(2.0 ** -100)) / np.float32(127.0)
    assert d.dtype == np.float32
    q = np.rint(z.astype(np.float64) / d.astype(np.float64)[:, None])
    return q.astype(np.int8), np.where(bad, np.float32(np.nan), d)


def i8_planes(q, d):
    """the I8_SPLIT bytes"""
    r, k = q.shape
    p = np.zeros((r, (k + 15) // 16 * 16), np.int8)
    p[:, :k] = q
    return np.concatenate([p.reshape(-1).view(np.uint8), np.ascontiguousarray(d, np.float32).view(np.uint8)])


def i8_unplanes(buf, rows, k):
    """integers with their padding (R, ld), scales"""
    ld = (k + 15) // 16 * 16
    return buf[:rows * ld].view(np.int8).reshape(rows, ld), buf[rows * ld:rows * (ld + 4)].view(np.float32)


def turn(x, pos, dims, halves, shared, base=10000.0, scale=1.0):
    """x (B, S, H, D), pos (B or 1, axes, S): the turned values and, for each value, |a| + |b| of its pair (0 where it is copied)"""
    x = np.asarray(x, np.float64)
    out, size, n, i = x.copy(), np.zeros_like(x), sum(dims), 0
    for a, k in enumerate(dims):
        for j in range(k // 2):
            f = np.longdouble(base) ** (np.longdouble(-2 * i) / n if shared else np.longdouble(-2 * j) / k) * np.longdouble(scale)
            t = np.asarray(pos, np.longdouble)[:, a] * f
            c, s = np.cos(t).astype(np.float64)[..., None], np.sin(t).astype(np.float64)[..., None]
            u, v = (i, n // 2 + i) if halves else (2 * i, 2 * i + 1)
            out[..., u], out[..., v] = x[..., u] * c - x[..., v] * s, x[..., u] * s + x[..., v] * c
            size[..., u] = size[..., v] = np.abs(x[..., u]) + np.abs(x[..., v])
            i += 1
    return out, size


def rms(x, w, eps):
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def attention(q, k, v, scale, count=None):
    """q (B, H, Nq, D), k / v (B, G, Nkv, D), count (B, Nkv) bool: o (B, Nq, H, D), sum p |v| / sum p of the same shape, and the
    largest scale |q| . |k| of each sequence and head"""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    B, H, Nq, D = q.shape
    o, size, big = np.zeros((B, Nq, H, D)), np.zeros((B, Nq, H, D)), 0.0
    for b in range(B):
        at = np.arange(k.shape[2]) if count is None else np.nonzero(count[b])[0]
        for h in range(H):
            g = h * k.shape[1] // H
            if not len(at):
                continue
            kk, vv = k[b, g, at], v[b, g, at]
            s = q[b, h] @ kk.T * scale
            big = max(big, float((np.abs(q[b, h]) @ np.abs(kk).T).max()) * scale)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            o[b, :, h], size[b, :, h] = p @ vv, p @ np.abs(vv)
    return o, size, big
