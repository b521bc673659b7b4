"""Cross attention whose weights meet V in two parts of k's type (PREC_F32), against 64 bits.

Tolerances, with A = sum p |v| / sum p of an output and the logits' and sums' terms of the one-part form (test_gpu_cross_attention):
- two parts lose 2^-16 (bf16: the rounding of what a rounding lost, 2^-8 each) or 2^-22 (f16) of a weight: U A; f16 parts below the
  normal numbers are off by up to 2^-25 of a weight of 1, which is at most twice the largest: Nkv 2^-24 max |v|. The sum adds the
  weights themselves, so nothing is lost below the line;
- a logit is a sum of D products in fp32, D 2^-23 scale |q| . |k|, times log2 e less the maximum, three more roundings of it, and its
  power of two is within 2^-22: a weight is off by 1.5 that, above and below the line;
- the sums over the states (two products each) and their rescaling: (2 Nkv + 64) 2^-23 A above the line, (Nkv + 64) 2^-23 A below it;
- the output's rounding, 2^-8, 2^-11 or 2^-24 of it."""
import numpy as np
import pytest

import crossref
from test_cross_ops_abi import cross_params
from test_gpu_cross_attention import SHAPES, U, host, shape, to  # noqa: F401  (shape: fixture)
from test_gpu_int8 import T  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu
TWO = {"bf16": 2.0 ** -16, "f16": 2.0 ** -22}


def tolerance(o, size, big, D, Nkv, kv, out, vmax):
    w = 1.5 * (big * (D + 3) * 2.0 ** -23 + 2.0 ** -22)
    tol = (TWO[kv] + 2 * w + (3 * Nkv + 128) * 2.0 ** -23) * size + (Nkv * 2.0 ** -24 * vmax if kv == "f16" else 0.0)
    return tol + U[out] * (np.abs(o) + tol) + (2.0 ** -24 if out == "f16" else 1e-37)


def check(T, q, k, v, kv, out="f32", count=None, scale=None, **kw):  # noqa: F811
    """held against 64 bits: the call in two parts, the same in one, and the 64-bit result"""
    (Q, q), (K, k), (V, v) = (to(T, t, kv) for t in (q, k, v))
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, size, big = crossref.attention(q, k, v, np.float32(scale), count)
    tol = tolerance(want, size, big, q.shape[-1], k.shape[2], kv, out, np.abs(v).max())
    two, one = (host(T.cross_attention(Q, K, V, scale=scale, out_dtype=out, prec=p, **kw)) for p in (T.PREC_F32, T.PREC_DEFAULT))
    assert np.isfinite(two).all()
    bad = np.abs(two - want) - tol
    assert bad.max() <= 0, (bad.max(), np.unravel_index(bad.argmax(), bad.shape))
    return two, one, want


@pytest.mark.parametrize("kv", ["bf16", "f16"])
@pytest.mark.parametrize("D", [24, 64, 72, 96, 128])
@pytest.mark.parametrize("rows,ranges", SHAPES)
def test_each_shape(T, shape, rows, ranges, D, kv):  # noqa: F811
    shape(rows, ranges)
    rng = np.random.default_rng(rows + D)
    q, k, v = (rng.standard_normal(s) for s in ((2, 6, 37, D), (2, 3, 1000, D), (2, 3, 1000, D)))
    lens = np.array([1000, 129], np.int32)
    two, one, want = check(T, q, k, v + 0.5, kv, count=np.arange(1000) < lens[:, None], kv_len=T.to_device(lens))
    # the one-part form's error is of its rounding's size (some 2^-9 or 2^-12 a weight, averaged): the two parts leave little of it
    assert np.linalg.norm(two - want) < (0.02 if kv == "bf16" else 0.1) * np.linalg.norm(one - want)
    flags = (rng.random((1, 777)) < 0.7).astype(np.uint8)
    q, k, v = (rng.standard_normal((1, 2, n, D)) * s for n, s in ((300, 3), (777, 1), (777, 1)))
    check(T, q, k, v, kv, kv, count=flags != 0, kv_valid=T.to_device(flags))


@pytest.mark.parametrize("kv", ["bf16", "f16"])
@pytest.mark.parametrize("rows,ranges", [(32, 1), (128, 1), (256, 1), (32, 16), (128, 16), (256, 16)])
def test_maximum_that_moves(T, shape, rows, ranges, kv):  # noqa: F811
    """logits that rise and fall past every threshold between and within ranges"""
    shape(rows, ranges)
    n, d, rng = 1500, 128, np.random.default_rng(3)
    for ramp in (np.linspace(0, 60, n), np.linspace(60, 0, n), np.linspace(-60, -50, n)):
        q = np.zeros((1, 1, 50, d), np.float32)
        q[..., 0] = 8.0 * np.linspace(-1, 1, 50)
        k = rng.standard_normal((1, 1, n, d)).astype(np.float32) * 0.1
        k[..., 0] = ramp
        check(T, q, k, rng.standard_normal((1, 1, n, d)), kv, scale=0.125)


def test_rows_that_nothing_counts_for(T):  # noqa: F811
    rng = np.random.default_rng(4)
    for nq in (1, 300):
        q, k, v = (to(T, rng.standard_normal((3, 2, n, 64)), "bf16")[0] for n in (nq, 200, 200))
        got = T.cross_attention(q, k, v, kv_len=T.to_device(np.array([0, 5, 0], np.int32)), prec=T.PREC_F32).numpy()
        assert (got[[0, 2]] == 0).all() and np.isfinite(got[1]).all() and (got[1] != 0).any()


def test_refusals(T):  # noqa: F811
    q = to(T, np.ones((1, 1, 3, 64)), "bf16")[0]
    for prec in (1, -1, 11):
        with pytest.raises(T.TskError, match="prec"):
            T.cross_attention(q, q, q, prec=prec)
    assert cross_params(T).prec == T.PREC_DEFAULT
