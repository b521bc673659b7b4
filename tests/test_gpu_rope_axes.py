"""Rotary positions over several axes on gfx950, against 64 bits.

Tolerances. Sines and cosines are off by at most 2^-22 (stated with the entry point), the two products and the sum of a
pair by 3 * 2^-24 of |a| + |b|: 2^-21 (|a| + |b|) together. The angle is formed in 64 bits: 2^-51 of itself. The norm of a head adds a sum
of squares in fp32 (8 products in a lane, then at most 6 sums of lanes), a mean, an eps, a root, a quotient and two
products: at most 24 roundings, 24 * 2^-24. Outputs of bf16 are off by 2^-8 of theirs, of f32 by 2^-24."""
import numpy as np
import pytest

import crossref
import mxref
from test_gpu_int8 import T, dev, host, typed  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def tolerance(x, size, want, far, norm, out_dtype):
    moved = np.where(size > 0, size, np.abs(x))
    tol = np.where(size > 0, 2.0 ** -21 + far * 2.0 ** -51, 0.0) * size + (24 * 2.0 ** -24 if norm else 0.0) * moved
    return tol + (2.0 ** -8 if out_dtype == "bf16" else 2.0 ** -24) * (np.abs(want) + tol) + 1e-37


def check(T, x, pos, dims, halves=False, shared=False, w=None, dtype="f32", out_dtype=None, base=10000.0, scale=1.0, eps=1e-6):  # noqa: F811
    out_dtype = out_dtype or dtype
    x = typed(x, dtype)
    X, P = dev(T, x, dtype), T.to_device(pos)
    out = dev(T, np.zeros(x.shape, np.float32), out_dtype)
    kw = dict(pairs=T.ROPE_HALVES if halves else T.ROPE_ADJACENT, shared_freqs=shared, freq_base=base, freq_scale=scale, eps=eps,
              w=None if w is None else T.to_device(w))
    got = host(T.rope_axes(X, P, dims, out=out, **kw))
    ref = x.astype(np.float64) if w is None else crossref.rms(x, w.astype(np.float64), np.float32(eps))
    want, size = crossref.turn(ref, pos if pos.ndim == 3 else pos[None], dims, halves, shared, np.float32(base), np.float32(scale))
    far = float(np.abs(pos.astype(np.float64)).max() * abs(scale))
    bad = np.abs(got - want) - tolerance(ref, size, want, far, w is not None, out_dtype)
    assert bad.max() <= 0, (bad.max(), np.unravel_index(bad.argmax(), bad.shape))
    if out_dtype == dtype:                                     # in place: the same bits
        T.rope_axes(X, P, dims, out=X, **kw)
        assert np.array_equal(host(X), got)


HEADS = [(64, (48, 16)), (64, (64,)), (128, (44, 42, 42)), (96, (32, 32, 32)), (72, (24, 24, 16)), (128, (16, 24, 24)),
         (33, (10, 6)), (2, (2,)), (8, (2, 2, 2, 2)), (130, (64, 0, 50)), (288, (64, 64, 64, 64)), (384, (126, 130, 128)), (17, (2,))]


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("halves,shared", [(False, False), (True, False), (True, True), (False, True)])
@pytest.mark.parametrize("d,dims", HEADS)
def test_heads(T, d, dims, halves, shared, norm):  # noqa: F811
    rng = np.random.default_rng(d)
    x = rng.standard_normal((2, 9, 5, d)).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(d)).astype(np.float32) if norm else None
    pos = rng.integers(-50, 2000, (2, len(dims), 9)).astype(np.int32)
    check(T, x, pos, dims, halves, shared, w)
    check(T, x, (rng.standard_normal((len(dims), 9)) * 300).astype(np.float32), dims, halves, shared, w, "bf16")


@pytest.mark.parametrize("b,s,h", [(1, 1, 1), (1, 1, 40), (3, 2, 7), (1, 700, 3), (2, 194, 16), (1, 5000, 1)])
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
def test_sizes_and_types(T, b, s, h, dtype, out):  # noqa: F811
    rng = np.random.default_rng(s)
    x = rng.standard_normal((b, s, h, 64)).astype(np.float32)
    check(T, x, rng.integers(0, 700, (b, 2, s)).astype(np.int32), (48, 16), w=np.ones(64, np.float32), dtype=dtype, out_dtype=out)


def test_far_positions(T):  # noqa: F811
    """positions past 2^24: the angle's last bits"""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((1, 6, 2, 32)).astype(np.float32)
    pos = np.array([[[2 ** 31 - 1, -2 ** 31, 16777217, 1 << 20, 0, -1]]], np.int32)
    check(T, x, pos, (32,))
    check(T, x, (pos * np.float32(1e3)).astype(np.float32), (32,), halves=True)


def test_bases_and_scales(T):  # noqa: F811
    rng = np.random.default_rng(5)
    x = rng.standard_normal((1, 20, 2, 64)).astype(np.float32)
    pos = np.stack([np.arange(20), np.zeros(20)]).astype(np.float32)
    for base, scale in ((1.0, 1.0), (500000.0, 0.125), (100.0, -2.5), (10000.0, 0.0), (0.5, 1.0)):
        check(T, x, pos, (32, 32), base=base, scale=scale)


def test_quarter_turns(T):  # noqa: F811
    """near multiples of a quarter turn the sine or cosine is small: it keeps its absolute accuracy"""
    x = np.ones((1, 64, 1, 2), np.float32)
    pos = (np.arange(64, dtype=np.float64) * np.pi / 2).astype(np.float32)[None]
    check(T, x, pos, (2,))


def test_positions_that_are_not_finite(T):  # noqa: F811
    x = np.ones((1, 4, 3, 16), np.float32)
    pos = np.array([[0, np.inf, 1, np.nan], [0, 1, -np.inf, 1]], np.float32)
    y = T.rope_axes(T.to_device(x), T.to_device(pos), (8, 4)).numpy()[0]
    assert np.isfinite(y[0]).all()
    assert np.isnan(y[[1, 3], :, :8]).all() and np.isfinite(y[[1, 3], :, 8:]).all()
    assert np.isnan(y[2, :, 8:12]).all() and np.isfinite(y[2, :, :8]).all() and (y[:, :, 12:] == 1).all()


def test_strided_views(T):  # noqa: F811
    """q and k as a projection leaves them, rows off 16 bytes, positions of every sequence in one array"""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((2, 11, 3, 4, 32)).astype(np.float32)
    for dtype in ("f32", "bf16"):
        X = dev(T, x, dtype)
        xt = typed(x, dtype)
        k = X.view(4 * 32, (2, 11, 4, 32), (11 * 384, 384, 32, 1))
        pos = T.to_device(rng.integers(0, 99, (2, 3, 16)).astype(np.int32))
        p = pos.view(2, (2, 3, 11), (48, 16, 1))
        T.rope_axes(k, p, (16, 8, 8), out=k)
        want, size = crossref.turn(xt[:, :, 1], pos.numpy()[:, :, 2:13], (16, 8, 8), False, False)
        got = host(X)
        assert (np.abs(got[:, :, 1] - want) - tolerance(xt[:, :, 1], size, want, 99, False, dtype)).max() <= 0
        assert np.array_equal(got[:, :, [0, 2]], xt[:, :, [0, 2]])
        odd = dev(T, x.reshape(2, 11, -1), dtype)
        o = odd.view(1, (2, 11, 4, 30), (11 * 384, 384, 31, 1))
        y = host(T.rope_axes(o, p, (10, 8, 8)))
        src = np.stack([typed(x, dtype).reshape(2, 11, -1)[..., 1 + 31 * h:31 + 31 * h] for h in range(4)], 2)
        want, size = crossref.turn(src, pos.numpy()[:, :, 2:13], (10, 8, 8), False, False)
        assert (np.abs(y - want) - tolerance(src, size, want, 99, False, dtype)).max() <= 0


def test_agrees_with_one_axis(T):  # noqa: F811
    """tsk_rope_ext on one axis, whose running product of the frequencies and fp32 angles are off by their own
    rounding: at most (pairs + 2) * 2^-24 of the angle"""
    rng = np.random.default_rng(7)
    x = rng.standard_normal((1, 100, 3, 64)).astype(np.float32)
    pos = np.arange(100, dtype=np.int32)
    a = T.rope_axes(T.to_device(x), T.to_device(pos[None]), (64,)).numpy()
    b = T.rope_ext(T.to_device(x), T.to_device(pos), 64).numpy()
    size = np.abs(x[..., 0::2]) + np.abs(x[..., 1::2])
    assert (np.abs(a - b).reshape(1, 100, 3, 32, 2).max(-1) <= size * (100 * 34 * 2.0 ** -24 + 2.0 ** -20)).all()


def test_replayed_from_a_graph(T):  # noqa: F811
    rng = np.random.default_rng(8)
    xs = [rng.standard_normal((2, 50, 4, 64)).astype(np.float32) for _ in range(3)]
    pos = T.to_device(rng.integers(0, 200, (2, 50)).astype(np.int32))
    want = [T.rope_axes(T.to_device(x), pos, (40, 24)).numpy() for x in xs]
    st, x, out = T.Stream(), T.to_device(xs[0]), T.to_device(np.zeros_like(xs[0]))
    T.synchronize()
    g = T.Graph(st, lambda: T.rope_axes(x, pos, (40, 24), out=out, stream=st))
    for i in (1, 2, 0):
        src = T.to_device(xs[i])
        T._hipcheck(T.hip().hipMemcpy(x.ptr, src.ptr, x.nbytes, 3), "hipMemcpy D2D")
        T.rope_axes(src, pos, (40, 24))
        T.synchronize()
        g.launch()
        st.synchronize()
        assert np.array_equal(out.numpy(), want[i])
    g.destroy()
    st.destroy()


@pytest.mark.parametrize("b,s,h", [(1, 2100, 70), (1, 9001, 3), (300, 10, 2), (1, 40, 200)])
@pytest.mark.parametrize("d,dims", [(64, (40, 24)), (65, (64,)), (20, (8, 6))])
@pytest.mark.parametrize("halves", [False, True])
def test_many(T, b, s, h, d, dims, halves):  # noqa: F811
    """more heads than are in flight at once, more tokens and sequences than waves, heads of a token over several waves"""
    rng = np.random.default_rng(h)
    x = rng.standard_normal((b, s, h, d)).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(d)).astype(np.float32)
    check(T, x, rng.integers(0, 3000, (b, len(dims), s)).astype(np.int32), dims, halves, w=w, dtype="bf16" if s > 2000 else "f32")
