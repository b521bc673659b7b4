"""MXFP4 products of more threads than one launch holds: the rounding of f32 activations and the product itself go in
pieces. Inputs are small integers times E2M1 numbers: sums are exact, results equal (in bf16 the sums rounded once)."""
import numpy as np
import pytest

import mxref
from test_gpu_mxfp4 import T, dev, operands, shape, split  # noqa: F401  (T, shape: fixtures)
from test_gpu_mxfp4_ends import fetch

pytestmark = pytest.mark.gpu


def test_rounding_of_activations(T):
    """2^21 + 9 rows of 8192 f32 values, four a thread: more than 2^32 threads; the rows overlap, each 4 values on"""
    rng = np.random.default_rng(1)
    n, k, m = (1 << 21) + 9, 8192, 16
    wc, wb, _, _ = operands(rng, 1, k, m, True)
    x = rng.integers(-8, 9, 4 * (n - 1) + k).astype(np.float32)
    xd = T.to_device(x)
    st, ws = T.Stream(), T.empty((n * k * 2 + 256,), "u8")
    out, W = T.empty((n, m)), split(T, wc, wb)
    T.synchronize()
    T.set_workspace(ws, stream=st)
    T.mul_mat(W, xd.view(0, (n, k), (4, 1)), out=out, stream=st)
    st.synchronize()
    T.set_workspace(None, stream=st)
    st.destroy()
    y, w = out.numpy(), mxref.values(wc, wb)
    for i in (0, 1, n // 2 - 1, n // 2, (1 << 20) - 1, 1 << 20, (1 << 20) + 1, (1 << 21) - 1, 1 << 21, n - 2, n - 1):
        assert np.array_equal(y[i], (w @ x[4 * i:4 * i + k]).astype(np.float32)), i


@pytest.mark.parametrize("act", ["mxfp4", "bf16"])
def test_product_in_two_launches(T, shape, act):
    """16 x 16 outputs a workgroup of 256 threads, 2^31 and more of them"""
    shape(11)
    rng = np.random.default_rng(2)
    n, k, m = (1 << 20) + 35, 32, 2050
    wc, wb, xc, xb = operands(rng, n, k, m, True)
    if act == "mxfp4":
        x, xd = None, split(T, xc, xb)
    else:
        x = rng.integers(-8, 9, (n, k)).astype(np.float32)
        xd = dev(T, x, act)
    out = T.empty((n, 2056), "bf16")
    T.mul_mat(split(T, wc, wb), xd, out=out.view(0, (n, m), (2056, 1)))
    half = (n // 2 + 15) // 16 * 16
    for i in (0, 17, half - 1, half, half + 1, half + 16, n - 2, n - 1):
        row = mxref.values(xc[i:i + 1], xb[i:i + 1]) if x is None else x[i:i + 1].astype(np.float64)
        want = mxref.bf16_bits((row @ mxref.values(wc, wb).T).astype(np.float32))[0]
        assert np.array_equal(fetch(T, out, i * 2056 * 2, (m,), np.uint16), want), i
