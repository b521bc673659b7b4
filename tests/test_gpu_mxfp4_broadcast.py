"""MXFP4 products and the quantizer on rows broadcast along one or two of their outer extents, as a conditioning row
expanded over its batch's tokens is. Inputs are small integers times E2M1 numbers: sums are exact, results equal."""
import numpy as np
import pytest

import mxref
from test_gpu_mxfp4 import T, dev, operands, split  # noqa: F401  (T: fixture)

pytestmark = pytest.mark.gpu

# extents (n3, n2, n1), and which of them are broadcast
VIEWS = [((1, 3, 5), "..b"), ((1, 3, 5), ".b."), ((2, 3, 4), "..b"), ((2, 3, 4), ".b."), ((2, 3, 4), "b.."), ((2, 3, 4), ".bb"),
         ((2, 3, 4), "bb."), ((2, 3, 4), "b.b"), ((3, 1, 4), "..b"), ((3, 1, 4), "b.."), ((3, 4, 1), ".b."), ((2, 3, 4), "bbb")]


def expanded(T, x, shape, dtype):
    """rows x of the extents that are not broadcast -> a view of shape + (K,), strides 0 where they are, and its values"""
    k = x.shape[-1]
    st, at = [], k
    for n, own in zip(shape[::-1], x.shape[-2::-1]):
        st.insert(0, at if own == n and n > 1 else 0)
        at *= own
    return dev(T, x, dtype).view(0, shape + (k,), tuple(st) + (1,)), np.broadcast_to(x, shape + (k,))


def rows_of(rng, shape, which, k):
    """integers, every row other than the others"""
    own = tuple(1 if w == "b" else n for n, w in zip(shape, which))
    return rng.integers(-8, 9, own + (k,)).astype(np.float32)


@pytest.mark.parametrize("shape,which", VIEWS)
@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_products(T, shape, which, act):
    rng = np.random.default_rng(sum(shape))
    k, m = 96, 40
    wc, wb, _, _ = operands(rng, 1, k, m, True)
    xd, x = expanded(T, rows_of(rng, shape, which, k), shape, act)
    want = (x.reshape(-1, k).astype(np.float64) @ mxref.values(wc, wb).T).astype(np.float32)
    assert np.array_equal(T.mul_mat(split(T, wc, wb), xd).numpy().reshape(-1, m), want)


@pytest.mark.parametrize("which", ["..b", ".b."])
@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_products_on_tiles(T, which, act):
    """300 rows a product: tiles, f32 rows rounded by a launch before"""
    rng = np.random.default_rng(11)
    shape, k, m = (1, 3, 300), 1024, 1024
    wc, wb, _, _ = operands(rng, 1, k, m, True)
    xd, x = expanded(T, rows_of(rng, shape, which, k), shape, act)
    want = (x.reshape(-1, k).astype(np.float64) @ mxref.values(wc, wb).T).astype(np.float32)
    assert np.array_equal(T.mul_mat(split(T, wc, wb), xd).numpy().reshape(-1, m), want)


@pytest.mark.parametrize("shape,which", VIEWS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantizer(T, shape, which, dtype):
    rng = np.random.default_rng(sum(shape))
    k = 64
    xd, x = expanded(T, rows_of(rng, shape, which, k), shape, dtype)
    assert np.array_equal(T.mxfp4_quantize(xd).buf.numpy(), mxref.planes(*mxref.quantize(np.ascontiguousarray(x.reshape(-1, k)))))
