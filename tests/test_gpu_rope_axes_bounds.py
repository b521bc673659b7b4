"""The header's bound of far angles: sines and cosines within 2^-22 + 2^-50 |freq_scale * position|, of bases below 1 within 2^-22 +
2^-46 |angle|. With u = 2^-53 the frequency's product of a constant, the scale and a power takes 4.6 u, its exponent |e| ln(base) u
and the product with the position 1 u: of the angle 5.6 u + |e| ln(base) u, which times a frequency base^e of at most 1 is at most
5.6 u; below 1, |e| |ln(base)| is at most 88. Values are 1 and 0 in turn, so that a pair's results are its cosine and sine, each
rounded once to fp32 (2^-24 of at most 1)."""
import numpy as np
import pytest

from test_gpu_int8 import T  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("base", [2.0, 1e4, 5e5, 1e9, 0.25, 1e-6])
@pytest.mark.parametrize("scale", [1.0, 0.3, -2.5])
@pytest.mark.parametrize("kind", ["i32", "f32"])
def test_far_angles(T, base, scale, kind):  # noqa: F811
    d, rng = 62, np.random.default_rng(1)
    far = np.array([2 ** 31 - 1, -2 ** 31, 1 << 30, 123456789, 3, 0])
    pos = far.astype(np.int32) if kind == "i32" else (far * 1000.0 + rng.random(6)).astype(np.float32)
    x = np.zeros((1, 6, 1, d), np.float32)
    x[..., 0::2] = 1
    got = T.rope_axes(T.to_device(x), T.to_device(pos[None]), (d,), freq_base=base, freq_scale=scale).numpy()[0, :, 0].astype(np.float64)
    f = np.longdouble(np.float32(base)) ** (np.arange(0, -d, -2).astype(np.longdouble) / d) * np.longdouble(np.float32(scale))
    t = pos.astype(np.longdouble)[:, None] * f
    tol = 2.0 ** -22 + 2.0 ** -24
    if base >= 1:
        tol = tol + 2.0 ** -50 * np.abs(pos.astype(np.float64) * np.float64(np.float32(scale)))[:, None]
    else:
        tol = tol + 2.0 ** -46 * np.abs(t).astype(np.float64)
    for i, fn in enumerate((np.cos, np.sin)):
        bad = np.abs(got[:, i::2] - fn(t).astype(np.float64)) - tol
        assert bad.max() <= 0, (bad.max(), np.unravel_index(bad.argmax(), bad.shape))


@pytest.mark.parametrize("base", [1.0, 1e4, 1e-6, 1e-38])
def test_the_farthest_angles(T, base):  # noqa: F811
    """angles past 2^53 quarter turns, up to those of the largest positions: still a cosine and a sine of one angle"""
    x = np.zeros((1, 130, 1, 16), np.float32)
    x[..., 0::2] = 1
    pos = (np.float32(2.0 ** 40) * np.exp2(np.arange(130) * 0.67) * np.where(np.arange(130) % 2, -1, 1)).astype(np.float32)
    assert np.isfinite(pos).all() and np.abs(pos).max() > 1e38
    for scale in (1.0, 0.37):
        y = T.rope_axes(T.to_device(x), T.to_device(pos[None]), (16,), freq_base=base, freq_scale=scale).numpy()[0, :, 0].astype(np.float64)
        assert np.abs(y[:, 0::2] ** 2 + y[:, 1::2] ** 2 - 1).max() <= 4 * 2.0 ** -22
