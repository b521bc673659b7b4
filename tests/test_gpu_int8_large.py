"""8-bit rows of the largest sizes: more threads than one launch holds (2^22 rows and more, of 1024 threads each; they overlap, each four
(f32) or eight (bf16) values on), and rows of nearly 2^31 values."""
import ctypes

import numpy as np
import pytest

import crossref
import mxref
from test_gpu_int8 import T, dev, off, planes, typed, want_linear  # noqa: F401  (T: fixture)
from test_gpu_mxfp4_ends import fetch

pytestmark = pytest.mark.gpu

N, K, LD = (1 << 22) + 37, 8200, 8208
ROWS = (0, 1, (1 << 20) - 1, 1 << 20, (1 << 21) + 3, (1 << 22) - 1, 1 << 22, N - 2, N - 1)


def rows(T, dtype):  # noqa: F811
    """the array, a row of it, and the view of all rows"""
    step = 4 if dtype == "f32" else 8
    x = typed(np.random.default_rng(3).standard_normal(step * (N - 1) + K).astype(np.float32), dtype)
    return lambda i: x[step * i:step * i + K][None], dev(T, x, dtype).view(0, (N, K), (step, 1))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize(T, dtype):  # noqa: F811
    row, x = rows(T, dtype)
    sp = T.i8_quantize(x)
    for i in ROWS:
        q, d = crossref.i8_quantize(row(i))
        assert np.array_equal(fetch(T, sp.buf, i * LD, (K,), np.int8), q[0]), i
        assert fetch(T, sp.buf, N * LD + 4 * i, (1,), np.float32) == d, i


def test_product(T):  # noqa: F811
    row, x = rows(T, "bf16")
    w = crossref.i8_quantize(np.random.default_rng(4).standard_normal((16, K)).astype(np.float32))
    st, out, ws = T.Stream(), T.empty((N, 16)), T.empty((N * (LD + 4) + 256,), "u8")
    W = planes(T, *w)
    T.synchronize()
    T.set_workspace(ws, stream=st)
    T.mul_mat(W, x, out=out, stream=st)
    st.synchronize()
    T.set_workspace(None, stream=st)
    st.destroy()
    y = out.numpy()
    for i in ROWS:
        want, tol = want_linear(crossref.i8_quantize(row(i)), w, None, "f32")
        assert off(y[i:i + 1], want, tol) <= 0, i


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_longest_row(T, dtype):  # noqa: F811
    """2^31 - 256 values, zeros but for runs at its start, past 2^30 and at its end, and back"""
    k, n, size = (1 << 31) - 256, 50000, 4 if dtype == "f32" else 2
    rng = np.random.default_rng(5)
    x = T.empty((1, k), dtype)
    T._hipcheck(T.hip().hipMemset(ctypes.c_void_p(x.ptr), 0, ctypes.c_size_t(x.nbytes)), "hipMemset")
    runs = [(at, typed(rng.standard_normal(n).astype(np.float32), dtype)) for at in (0, (1 << 30) - 17, k - n)]
    for at, v in runs:
        src = np.ascontiguousarray(v if dtype == "f32" else mxref.bf16_bits(v))
        T._hipcheck(T.hip().hipMemcpy(ctypes.c_void_p(x.ptr + at * size), ctypes.c_void_p(src.ctypes.data), ctypes.c_size_t(src.nbytes), 1),
                    "hipMemcpy H2D")
    sp = T.i8_quantize(x)
    q, d = crossref.i8_quantize(np.concatenate([v for _, v in runs])[None])
    assert fetch(T, sp.buf, k, (1,), np.float32) == d
    back = T.i8_dequantize(sp, dtype, out=x)
    for i, (at, _) in enumerate(runs):
        want = q[0, i * n:(i + 1) * n]
        assert np.array_equal(fetch(T, sp.buf, at, (n,), np.int8), want), at
        got = fetch(T, back, at * size, (n,), np.float32 if dtype == "f32" else np.uint16)
        value = want.astype(np.float32) * d
        assert np.array_equal(got, value if dtype == "f32" else mxref.bf16_bits(value).reshape(-1)), at
        if at:
            assert not fetch(T, sp.buf, at - n, (n,), np.int8).any(), at
