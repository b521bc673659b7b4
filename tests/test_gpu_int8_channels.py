"""Few rows of activations times 8-bit weights of very many channels: quantized in a launch of their own or inside the product,
the same bits."""
import ctypes

import numpy as np
import pytest

import crossref
from test_gpu_int8 import T, dev, off, planes, typed, want_linear  # noqa: F401  (T: fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("n,k,m", [(1, 256, 32768), (1, 256, 32784), (4, 200, 40000), (1, 2048, 40000), (2, 2048, 32776), (3, 77, 152064)])
def test_bits_of_every_way(T, n, k, m, act):  # noqa: F811
    rng = np.random.default_rng(m)
    x = typed((rng.standard_normal((n, k)) * np.exp(rng.standard_normal((n, 1)))).astype(np.float32), act)
    w = crossref.i8_quantize((rng.standard_normal((m, k)) * np.exp(rng.standard_normal((m, 1)))).astype(np.float32))
    pad = np.zeros((n, (k + 7) // 8 * 8), np.float32)
    pad[:, :k] = x
    X, W = dev(T, pad, act).view(0, (n, k), (pad.shape[1], 1)), planes(T, *w)
    got = T.mul_mat(W, X).numpy()
    want, tol = want_linear(crossref.i8_quantize(x), w, None, "f32")
    assert off(got, want, tol) <= 0
    assert np.array_equal(T.mul_mat(W, T.i8_quantize(X)).numpy(), got)
    # a capture on a stream without scratch, which cannot be had then, replayed between eager work
    st, out = T.Stream(), T.empty((n, m))
    T.synchronize()
    g = T.Graph(st, lambda: T.mul_mat(W, X, out=out, stream=st))
    for _ in range(3):
        T._hipcheck(T.hip().hipMemset(ctypes.c_void_p(out.ptr), 255, out.nbytes), "hipMemset")
        T.mul_mat(W, X)
        T.synchronize()
        g.launch()
        st.synchronize()
        assert np.array_equal(out.numpy(), got)
    g.destroy()
    st.destroy()
