"""8-bit rows and products at the ends of fp32's range."""
import numpy as np
import pytest

import crossref
from test_gpu_int8 import T, check_planes, dev, planes  # noqa: F401  (T: fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [5, 64, 1000, 20000])
def test_the_largest_numbers(T, k):  # noqa: F811
    """rows filled with the type's lowest number, and with the one above it: 127 d passes fp32's largest for the first alone"""
    low = np.finfo(np.float32).min
    x = np.random.default_rng(k).standard_normal((4, k)).astype(np.float32)
    x[0], x[1, 0], x[2], x[3, k - 1] = low, low, np.nextafter(low, np.float32(0)), -low
    sp = T.i8_quantize(dev(T, x))
    check_planes(sp, x, k)
    y = T.i8_dequantize(sp).numpy()
    assert np.isneginf(y[0]).all() and np.isneginf(y[1, 0]) and np.isposinf(y[3, k - 1])
    assert np.isfinite(y[2]).all() and np.isfinite(y[1, 1:]).all() and np.isfinite(y[3, :-1]).all()


def test_products_of_the_largest_rows(T):  # noqa: F811
    """sums are exact whatever the rows' size; then the token's scale, then the channel's"""
    rng, k = np.random.default_rng(1), 300
    x = crossref.i8_quantize((rng.standard_normal((20, k)) * 2.0 ** 100).astype(np.float32))
    w = crossref.i8_quantize((rng.standard_normal((16, k)) * 2.0 ** -110).astype(np.float32))
    got = T.mul_mat(planes(T, *w), planes(T, *x)).numpy()
    acc = x[0].astype(np.int64) @ w[0].astype(np.int64).T
    want = (acc.astype(np.float32) * x[1][:, None]) * w[1][None]
    assert np.isfinite(got).all() and np.array_equal(got, want)
