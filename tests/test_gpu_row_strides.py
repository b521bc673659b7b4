"""Products whose rows lie along the outermost extent, with gaps between its items or broadcast over it, the extent between
having one element: the items' own rows, whatever that extent's stride says. Inputs are small integers: F32 and BF16
weights give equal results; Q8_0 weights and rows of values up to 127 with one of 127 in every block (scale 1) too."""
import numpy as np
import pytest

import mxref
from test_gpu_mxfp4 import T  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def weights(T, rng, kind, m, k):
    w = rng.integers(-8, 9, (m, k)).astype(np.float32)
    if kind == "q8_0":
        w[:, ::32] = 127.0
        return w, T.q8_0_quantize(T.to_device(w)), T.Q8_0
    return w, T.to_device(w) if kind == "f32" else T.bf16_to_device(mxref.bf16_bits(w)), None


@pytest.mark.parametrize("kind", ["f32", "bf16", "q8_0"])
@pytest.mark.parametrize("n", [1, 2, 6, 70])
@pytest.mark.parametrize("between", [0, 1, 2])
def test_items_apart(T, kind, n, between):
    """[K, n, 1, 3] out of [K, n + 4, 1, 3]; the stride of the extent of 1: one item's, its rows', none"""
    rng = np.random.default_rng(n)
    k, m = 128, 48
    w, wd, at = weights(T, rng, kind, m, k)
    x = rng.integers(-8, 9, (3, n + 4, k)).astype(np.float32)
    x[:, :, ::32] = 127.0
    gap = (n + 4) * k
    v = T.to_device(x).view(0, (3, 1, n, k), (gap, (gap, n * k, 0)[between], k, 1))
    out = T.to_device(np.full((3, n + 2, m), 5.0, np.float32))
    og = (n + 2) * m
    T.mul_mat(wd, v, out=out.view(0, (3, 1, n, m), (og, (og, n * m, 0)[between], m, 1)), a_type=at)
    got = out.numpy()
    assert np.array_equal(got[:, :n], (x[:, :n].astype(np.float64) @ w.T.astype(np.float64)).astype(np.float32))
    assert (got[:, n:] == 5.0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "q8_0"])
@pytest.mark.parametrize("n", [2, 6, 70])
def test_items_broadcast(T, kind, n):
    """the same n rows for every item"""
    rng = np.random.default_rng(n)
    k, m = 128, 48
    w, wd, at = weights(T, rng, kind, m, k)
    x = rng.integers(-8, 9, (n, k)).astype(np.float32)
    x[:, ::32] = 127.0
    got = T.mul_mat(wd, T.to_device(x).view(0, (3, 1, n, k), (0, 0, k, 1)), a_type=at).numpy()
    want = (x.astype(np.float64) @ w.T.astype(np.float64)).astype(np.float32)
    assert np.array_equal(got, np.broadcast_to(want, (3, 1, n, m)))
