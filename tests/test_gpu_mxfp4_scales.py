"""MXFP4 products at the ends of the scale. A weight of 2^128 or more is infinite next to bf16 activations (bf16 and f32
hold no more; 0 times it is NaN), and exact next to MXFP4 ones, whose codes and scales are multiplied apart; the
smallest, 2^-128, is exact next to both. One product a result, the other terms 0: results equal."""
import numpy as np
import pytest

import mxref
from test_gpu_mxfp4 import T, dev, shape, split  # noqa: F401  (T, shape: fixtures)

pytestmark = pytest.mark.gpu
BYTES = [0, 1, 2, 3, 126, 127, 128, 135, 200, 251, 252, 253, 254]
AT = 37                                                        # where rows of either operand are not 0


def weights(k):
    """a row for every scale byte and number, its value at AT"""
    codes, byte = np.zeros((len(BYTES) * 16, k), np.uint8), np.full((len(BYTES) * 16, k // 32), 127, np.uint8)
    codes[:, AT], byte[:, AT // 32] = np.tile(np.arange(16), len(BYTES)), np.repeat(BYTES, 16)
    return codes, byte


@pytest.mark.parametrize("cfg", [0, 3, 4, 5, 9, 11, 14])
@pytest.mark.parametrize("act", ["bf16", "f32", "mxfp4"])
def test_every_number(T, shape, cfg, act):
    """the activation's power of two brings the product back into fp32's normal range: rows by launch shape"""
    shape(cfg)
    k = 128
    wc, wb = weights(k)
    w = mxref.values(wc, wb)[:, AT]
    powers = [-110, -60, -3, 0, 5, 70, 120]
    for n in (len(powers), 70):
        e = np.array((powers * 70)[:n])
        if act == "mxfp4":
            xc, xb = np.zeros((n, k), np.uint8), np.full((n, k // 32), 127, np.uint8)
            xc[:, AT], xb[:, AT // 32] = 2, 127 + e            # 1.0 times 2^e
            xd = split(T, xc, xb)
        else:
            x = np.zeros((n, k), np.float32)
            x[:, AT] = 2.0 ** e
            xd = dev(T, x, act)
            with np.errstate(over="ignore"):
                w = w.astype(np.float32).astype(np.float64)    # 2^128 up: infinite
        p = 2.0 ** e[:, None] * w[None, :]
        y = T.mul_mat(split(T, wc, wb), xd).numpy()
        normal = (np.abs(p) >= 2.0 ** -126) | (p == 0)         # (smaller ones may be flushed)
        with np.errstate(over="ignore"):
            want = p.astype(np.float32)
        assert np.array_equal(y[normal], want[normal]), n
        assert (np.abs(y[~normal]) <= np.abs(want[~normal])).all()


@pytest.mark.parametrize("act", ["bf16", "mxfp4"])
@pytest.mark.parametrize("n", [3, 70])
def test_zero_activations(T, act, n):
    """0 times a weight: 0, but NaN where next to bf16 the weight is infinite"""
    k = 128
    wc, wb = weights(k)
    y = T.mul_mat(split(T, wc, wb), dev(T, np.zeros((n, k), np.float32), "bf16") if act == "bf16" else
                  split(T, np.zeros((n, k), np.uint8), np.full((n, k // 32), 127, np.uint8))).numpy()
    infinite = np.abs(mxref.values(wc, wb)[:, AT]) >= 2.0 ** 128
    assert infinite.sum() == 2 * (2 + 4)                        # 4 and 6 times 2^126; 2, 3, 4 and 6 times 2^127
    want = np.where(infinite, np.nan, 0.0) if act == "bf16" else np.zeros(len(wc))
    assert np.array_equal(y, np.tile(want.astype(np.float32), (n, 1)), equal_nan=True)
