"""Cross attention on gfx950, against 64 bits.

Tolerances, with A = sum p |v| / sum p of an output and u = 2^-8 (bf16) or 2^-11 (f16), half a step of k's type:
- the weights are rounded to k's type, above and below the line: 2 u A; f16 weights below its normal numbers are off by up to 2^-25
  of the largest weight each instead, which is at most the sum: Nkv 2^-24 max |v|;
- a logit is a sum of D products in fp32, D 2^-23 scale |q| . |k| (truncation allowed for), times log2 e less the maximum, three more
  roundings of it, and its power of two is within 2^-22: a weight is off by 1.5 that, above and below the line;
- the sums over the states and their rescaling: (Nkv + 64) 2^-23 A, twice;
- the output's rounding, 2^-8, 2^-11 or 2^-24 of it."""
import numpy as np
import pytest

import crossref
import mxref
from test_gpu_int8 import T  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def to(T, x, dtype):  # noqa: F811
    """on the device in a type, and its values"""
    if dtype == "bf16":
        b = mxref.bf16_bits(np.asarray(x, np.float32))
        return T.bf16_to_device(b), mxref.bf16_values(b).reshape(np.shape(x))
    y = np.asarray(x, np.float16 if dtype == "f16" else np.float32)
    return T.to_device(y), y.astype(np.float32)


def host(a):
    return mxref.bf16_values(a.numpy()) if a.dtype == "bf16" else a.numpy().astype(np.float32)


def tolerance(o, size, big, D, Nkv, kv, out, vmax):
    w = 1.5 * (big * (D + 3) * 2.0 ** -23 + 2.0 ** -22)
    tol = (2 * U[kv] + 2 * w + 2 * (Nkv + 64) * 2.0 ** -23) * size + (Nkv * 2.0 ** -24 * vmax if kv == "f16" else 0.0)
    return tol + U[out] * (np.abs(o) + tol) + (2.0 ** -24 if out == "f16" else 1e-37)


def check(T, rng, B, H, G, Nq, Nkv, D, kv="bf16", qt=None, out=None, kv_len=None, valid=None, q_len=None, scale=None, spread=1.0):  # noqa: F811
    qt, out = qt or kv, out or kv
    Q, q = to(T, rng.standard_normal((B, H, Nq, D)) * spread, qt)
    K, k = to(T, rng.standard_normal((B, G, Nkv, D)), kv)
    V, v = to(T, rng.standard_normal((B, G, Nkv, D)) + 0.5, kv)
    count = None
    if kv_len is not None:
        count = np.arange(Nkv) < np.asarray(kv_len)[:, None]
    if valid is not None:
        flags = np.broadcast_to(valid != 0, (B, Nkv))
        count = flags if count is None else count & flags
    O, _ = to(T, np.full((B, Nq, H, D), 77.0), out)
    i32 = lambda t: None if t is None else T.to_device(np.asarray(t, np.int32))
    scale = D ** -0.5 if scale is None else scale
    T.cross_attention(Q, K, V, scale=scale, kv_len=i32(kv_len), q_len=i32(q_len),
                      kv_valid=None if valid is None else T.to_device(np.ascontiguousarray(valid, np.uint8)), out=O)
    got = host(O)
    q = to(T, q, kv)[1]                                        # (q is converted to k's type)
    want, size, big = crossref.attention(q, k, v, np.float32(scale), count)
    tol = tolerance(want, size, big, D, Nkv, kv, out, np.abs(v).max())
    if q_len is not None:
        behind = np.arange(Nq) >= np.asarray(q_len)[:, None]
        assert (got[behind] == 77.0).all()
        got[behind] = want[behind]
    assert np.isfinite(got).all()
    bad = np.abs(got - want) - tol
    assert bad.max() <= 0, (bad.max(), np.unravel_index(bad.argmax(), bad.shape))
    if count is not None:
        none = ~count.any(1)
        if q_len is None:
            assert (got[none] == 0).all()
    return O


SIZES = [(1, 1, 1, 1, 1, 64), (1, 1, 1, 1, 1, 8), (2, 3, 3, 5, 7, 64), (1, 16, 16, 646, 77, 64), (2, 4, 2, 33, 64, 128), (1, 8, 1, 1, 300, 128),
         (3, 6, 2, 31, 65, 96), (1, 2, 2, 128, 1000, 72), (2, 2, 1, 129, 127, 40), (1, 2, 2, 200, 2049, 128), (1, 32, 8, 1, 5000, 128),
         (4, 4, 4, 2, 4100, 64), (1, 1, 1, 700, 640, 120), (1, 5, 5, 257, 192, 16), (1, 1, 1, 3, 20000, 64), (2, 1, 1, 1030, 130, 128)]


@pytest.mark.parametrize("kv", ["bf16", "f16"])
@pytest.mark.parametrize("B,H,G,Nq,Nkv,D", SIZES)
def test_sizes(T, B, H, G, Nq, Nkv, D, kv):  # noqa: F811
    check(T, np.random.default_rng(Nq + Nkv), B, H, G, Nq, Nkv, D, kv)


@pytest.mark.parametrize("kv", ["bf16", "f16"])
@pytest.mark.parametrize("qt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
def test_types(T, kv, qt, out):  # noqa: F811
    check(T, np.random.default_rng(1), 1, 4, 2, 40, 100, 64, kv, qt, out)
    check(T, np.random.default_rng(2), 1, 4, 2, 3, 900, 104, kv, qt, out)


@pytest.mark.parametrize("Nq,Nkv,D", [(1, 200, 64), (70, 200, 128), (3, 3000, 64), (200, 3000, 128), (40, 64, 80)])
def test_lengths(T, Nq, Nkv, D):  # noqa: F811
    """none, one, a whole tile, one more, all, and those that are clamped"""
    lens = [0, 1, 64, 65, Nkv - 1, Nkv, Nkv + 5, -3, 128]
    check(T, np.random.default_rng(Nkv), len(lens), 2, 1, Nq, Nkv, D, kv_len=lens)
    check(T, np.random.default_rng(Nkv), len(lens), 2, 2, Nq, Nkv, D, "f16", kv_len=lens,
          q_len=[0, 1, Nq, Nq // 2, Nq, 5, 33, Nq + 9, -1])
    check(T, np.random.default_rng(Nkv), 3, 4, 2, Nq, Nkv, D, q_len=[0, Nq // 2 + 1, Nq])


@pytest.mark.parametrize("Nq,Nkv,D", [(1, 200, 64), (70, 200, 128), (3, 3000, 64), (200, 3000, 128), (40, 64, 80)])
def test_flags(T, Nq, Nkv, D):  # noqa: F811
    """single states, whole tiles and everything left out; flags other than 1; one set of flags for all; lengths beside them"""
    rng = np.random.default_rng(Nkv)
    v = (rng.random((6, Nkv)) < 0.6).astype(np.uint8) * rng.integers(1, 256, (6, Nkv)).astype(np.uint8)
    v[1] = 0
    v[2, :64] = 0
    v[3] = 0
    v[3, Nkv - 1] = 128
    v[4] = 1
    check(T, rng, 6, 2, 1, Nq, Nkv, D, valid=v)
    check(T, rng, 6, 2, 2, Nq, Nkv, D, "f16", valid=v, kv_len=[Nkv, 3, 64, Nkv - 1, 100, 30])
    check(T, rng, 3, 2, 2, Nq, Nkv, D, valid=v[5])


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
@pytest.mark.parametrize("Nq,Nkv,D", [(1, 300, 64), (70, 300, 128), (2, 4000, 128), (150, 100, 72)])
def test_what_does_not_count_has_no_effect(T, Nq, Nkv, D, bad):  # noqa: F811
    """the same bits whatever the states past the length or without their flag hold"""
    rng = np.random.default_rng(9)
    B = 2
    lens, flags = np.array([Nkv // 2 + 3, Nkv - 2], np.int32), (rng.random((B, Nkv)) < 0.7).astype(np.uint8)
    q = to(T, rng.standard_normal((B, 2, Nq, D)), "bf16")[0]
    k, v = (rng.standard_normal((B, 2, Nkv, D)).astype(np.float32) for _ in range(2))
    for use_len, use_flags in ((True, False), (False, True), (True, True)):
        count = np.ones((B, Nkv), bool)
        if use_len:
            count &= np.arange(Nkv) < lens[:, None]
        if use_flags:
            count &= flags != 0
        kw = dict(kv_len=T.to_device(lens) if use_len else None, kv_valid=T.to_device(flags) if use_flags else None, out_dtype="bf16")
        want = host(T.cross_attention(q, to(T, k, "bf16")[0], to(T, v, "bf16")[0], **kw))
        hole = ~np.broadcast_to(count[:, None, :, None], k.shape)
        for kk, vv in ((np.where(hole, np.float32(bad), k), v), (k, np.where(hole, np.float32(bad), v)),
                       (np.where(hole, np.float32(bad), k), np.where(hole, np.float32(bad), v))):
            got = host(T.cross_attention(q, to(T, kk, "bf16")[0], to(T, vv, "bf16")[0], **kw))
            assert np.isfinite(got).all() and np.array_equal(got, want)


def test_states_that_count_and_are_not_finite(T):  # noqa: F811
    """they reach the tokens of their sequence and head, no others"""
    rng = np.random.default_rng(11)
    q, k, v = (rng.standard_normal((2, 2, n, 64)).astype(np.float32) for n in (40, 90, 90))
    v[1, 0, 70, 5] = np.nan
    k[0, 1, 3, 0] = np.nan
    o = host(T.cross_attention(*(to(T, t, "bf16")[0] for t in (q, k, v)), out_dtype="f32"))
    assert np.isnan(o[1, :, 0, 5]).all() and np.isnan(o[0, :, 1]).all()
    assert np.isfinite(o[0, :, 0]).all() and np.isfinite(o[1, :, 1]).all() and np.isfinite(np.delete(o[1, :, 0], 5, -1)).all()


@pytest.mark.parametrize("kv", ["bf16", "f16"])
@pytest.mark.parametrize("spread", [0.0, 8.0, 40.0])
def test_flat_and_sharp_weights(T, kv, spread):  # noqa: F811
    rng = np.random.default_rng(3)
    check(T, rng, 1, 2, 2, 70, 500, 64, kv, spread=spread)
    check(T, rng, 1, 2, 2, 1, 5000, 128, kv, spread=spread)
    check(T, rng, 1, 2, 2, 64, 300, 64, kv, scale=3.0, spread=spread / 8)


@pytest.mark.parametrize("order", ["rising", "falling"])
def test_maximum_that_moves(T, order):  # noqa: F811
    """logits that rise from state to state past every threshold, and the other way round"""
    n, d = 1000, 64
    rng = np.random.default_rng(13)
    ramp = np.linspace(0, 60, n) if order == "rising" else np.linspace(60, 0, n)
    q = np.zeros((1, 1, 33, d), np.float32)
    q[..., 0] = 8.0 * np.linspace(-1, 1, 33)
    k = rng.standard_normal((1, 1, n, d)).astype(np.float32) * 0.1
    k[..., 0] = ramp
    v = rng.standard_normal((1, 1, n, d)).astype(np.float32)
    for kv in ("bf16", "f16"):
        (Q, q2), (K, k2), (V, v2) = (to(T, t, kv) for t in (q, k, v))
        got = T.cross_attention(Q, K, V, scale=0.125).numpy()
        want, size, big = crossref.attention(q2, k2, v2, 0.125)
        assert (np.abs(got - want) - tolerance(want, size, big, d, n, kv, "f32", np.abs(v2).max())).max() <= 0


def test_strided_views_and_shared_states(T):  # noqa: F811
    """q, k and v side by side in rows of a projection; one set of states for all sequences; an output with gaps"""
    rng = np.random.default_rng(5)
    B, N, M, H, D = 3, 50, 90, 4, 64
    X, x = to(T, rng.standard_normal((B, N, H, D)), "bf16")
    KV, kv = to(T, rng.standard_normal((1, M, 2, H, D)), "bf16")
    q = X.view(0, (B, H, N, D), (N * H * D, D, H * D, 1))
    k, v = (KV.view(i * H * D, (B, H, M, D), (0, D, 2 * H * D, 1)) for i in (0, 1))
    O, _ = to(T, np.full((B, N, H, 80), 5.0), "f32")
    lens = np.array([90, 40, 0], np.int32)
    T.cross_attention(q, k, v, kv_len=T.to_device(lens), out=O.view(8, (B, N, H, D), O.strides))
    kk, vv = (np.broadcast_to(kv[:, :, i].transpose(0, 2, 1, 3), (B, H, M, D)) for i in (0, 1))
    want, size, big = crossref.attention(x.transpose(0, 2, 1, 3), kk, vv, 0.125, np.arange(M) < lens[:, None])
    got = O.numpy()
    assert (np.abs(got[..., 8:72] - want) - tolerance(want, size, big, D, M, "bf16", "f32", np.abs(vv).max())).max() <= 0
    assert (got[..., :8] == 5.0).all() and (got[..., 72:] == 5.0).all()


def test_far_states(T):  # noqa: F811
    """states whose offsets pass 2^31 bytes: rows 2^20 bytes apart"""
    rng = np.random.default_rng(6)
    n, d, step = 4200, 64, 1 << 19
    big = T.empty(((n - 1) * step + 2 * d,), "bf16")
    k, v = (rng.standard_normal((n, d)).astype(np.float32) for _ in range(2))
    both = mxref.bf16_bits(np.concatenate([k, v], 1))
    H = T.hip()
    H.hipMemcpy2D.argtypes = [np.ctypeslib.ctypes.c_void_p, np.ctypeslib.ctypes.c_size_t] * 2 + [np.ctypeslib.ctypes.c_size_t] * 2 + [
        np.ctypeslib.ctypes.c_int]
    T._hipcheck(H.hipMemcpy2D(big.ptr, 2 * step, both.ctypes.data, 4 * d, 4 * d, n, 1), "hipMemcpy2D")
    K, V = (big.view(i * d, (1, 1, n, d), (0, 0, step, 1)) for i in (0, 1))
    for nq in (1, 130):
        Q, q = to(T, rng.standard_normal((1, 1, nq, d)), "bf16")
        got = T.cross_attention(Q, K, V).numpy()
        kk, vv = (mxref.bf16_values(mxref.bf16_bits(t))[None, None] for t in (k, v))
        want, size, big_ = crossref.attention(q, kk, vv, 0.125)
        assert (np.abs(got - want) - tolerance(want, size, big_, d, n, "bf16", "f32", np.abs(vv).max())).max() <= 0


@pytest.mark.parametrize("B,H,G,Nq,Nkv,D", [(2, 4, 2, 1, 3000, 128), (1, 2, 2, 100, 200, 64), (1, 1, 1, 40, 9000, 64)])
def test_bits_of_every_call(T, B, H, G, Nq, Nkv, D):  # noqa: F811
    """the same bits eager, on another stream with a bound workspace, and replayed from a graph between eager work"""
    import ctypes

    rng = np.random.default_rng(Nkv)
    qs = [to(T, rng.standard_normal((B, H, Nq, D)), "bf16")[0] for _ in range(3)]
    K, V = (to(T, rng.standard_normal((B, G, Nkv, D)), "bf16")[0] for _ in range(2))
    want = [T.cross_attention(q, K, V).numpy() for q in qs]
    assert np.array_equal(T.cross_attention(qs[0], K, V).numpy(), want[0])
    st, q, out = T.Stream(), T.empty((B, H, Nq, D), "bf16"), T.to_device(np.zeros((B, Nq, H, D), np.float32))
    need = T.workspace_size(T.OP_CROSS_ATTENTION, [q, K, V], out)
    ws = T.empty((max(need, 256),), "u8")
    T.set_workspace(ws, st)
    T.synchronize()
    g = T.Graph(st, lambda: T.cross_attention(q, K, V, out=out, stream=st))
    for i in (1, 2, 0, 1):
        T._hipcheck(T.hip().hipMemcpy(ctypes.c_void_p(q.ptr), ctypes.c_void_p(qs[i].ptr), q.nbytes, 3), "hipMemcpy D2D")
        T.cross_attention(qs[0], K, V)
        T.synchronize()
        g.launch()
        st.synchronize()
        assert np.array_equal(out.numpy(), want[i])
    g.destroy()
    st.synchronize()
    T.set_workspace(None, st)
    st.destroy()


@pytest.mark.parametrize("Nkv", [100, 3000])
def test_two_streams(T, Nkv):  # noqa: F811
    """calls on two streams keep to their own scratch"""
    rng = np.random.default_rng(1)
    K, V = (to(T, rng.standard_normal((1, 2, Nkv, 64)), "bf16")[0] for _ in range(2))
    qs = [to(T, rng.standard_normal((1, 2, n, 64)), "bf16")[0] for n in (1, 40)]
    want = [T.cross_attention(q, K, V).numpy() for q in qs]
    st, outs = [T.Stream(), T.Stream()], [T.empty(w.shape) for w in want]
    T.synchronize()
    for _ in range(20):
        for s, q, o in zip(st, qs, outs):
            T.cross_attention(q, K, V, out=o, stream=s)
    for s in st:
        s.synchronize()
    for o, w in zip(outs, want):
        assert np.array_equal(o.numpy(), w)
    for s in st:
        s.destroy()


@pytest.fixture
def shape(T, monkeypatch):  # noqa: F811
    """every call with one shape: rows of a workgroup and ranges of the states"""
    def use(rows, ranges):
        monkeypatch.setenv("TSK_CROSS_CFG", str(100 * rows + ranges))
        T.init(0, reread=True)
    yield use
    monkeypatch.delenv("TSK_CROSS_CFG", raising=False)
    T.init(0, reread=True)


SHAPES = [(r, n) for r in (32, 128, 256) for n in (1, 2, 16, 64)]


@pytest.mark.parametrize("D", [24, 32, 40, 64, 72, 96, 104, 128])
@pytest.mark.parametrize("rows,ranges", SHAPES)
def test_each_shape(T, shape, rows, ranges, D):  # noqa: F811
    """shared heads whose number is no multiple of 8, few heads, ragged rows and tiles, lengths that leave ranges empty"""
    shape(rows, ranges)
    rng = np.random.default_rng(rows + D)
    check(T, rng, 3, 6, 3, 37, 1000, D, kv_len=[1000, 129, 0], spread=3.0)
    check(T, rng, 1, 10, 10, 33, 130, D, kv="f16", out="f32", spread=3.0)
    check(T, rng, 1, 2, 2, 300, 777, D, valid=(rng.random((1, 777)) < 0.7), q_len=[290])
    check(T, rng, 2, 1, 1, 1, 64 * ranges + 1, D, kv="f16", kv_len=[64 * ranges + 1, 1], valid=np.arange(64 * ranges + 1) != 5)


@pytest.mark.parametrize("rows,ranges", SHAPES)
def test_maximum_that_moves_in_each_shape(T, shape, rows, ranges):  # noqa: F811
    """logits that rise, fall and jump past every threshold between and within ranges"""
    shape(rows, ranges)
    n, d, rng = 1500, 128, np.random.default_rng(3)
    jump = np.zeros(n)
    jump[::97] = np.linspace(10, 60, len(jump[::97]))
    for ramp in (np.linspace(0, 60, n), np.linspace(60, 0, n), jump, np.linspace(-60, -50, n)):
        q = np.zeros((1, 1, 50, d), np.float32)
        q[..., 0] = 8.0 * np.linspace(-1, 1, 50)
        k = rng.standard_normal((1, 1, n, d)).astype(np.float32) * 0.1
        k[..., 0] = ramp
        v = rng.standard_normal((1, 1, n, d)).astype(np.float32)
        for kv in ("bf16", "f16"):
            (Q, q2), (K, k2), (V, v2) = (to(T, t, kv) for t in (q, k, v))
            got = T.cross_attention(Q, K, V, scale=0.125).numpy()
            want, size, big = crossref.attention(q2, k2, v2, 0.125)
            assert (np.abs(got - want) - tolerance(want, size, big, d, n, kv, "f32", np.abs(v2).max())).max() <= 0


@pytest.mark.parametrize("rows,ranges", SHAPES)
def test_states_that_do_not_count_in_each_shape(T, shape, rows, ranges):  # noqa: F811
    """NaN and infinities where no state counts; a NaN that counts reaches its rows and no others"""
    shape(rows, ranges)
    rng = np.random.default_rng(9)
    B, Nq, n, d = 2, 40, 400, 64
    q, k, v = (rng.standard_normal((B, 1, m, d)).astype(np.float32) for m in (Nq, n, n))
    lens = np.array([333, 150], np.int32)
    for b in range(B):
        k[b, 0, lens[b]:] = np.nan
        v[b, 0, lens[b]:] = np.inf
    flags = np.ones((B, n), np.uint8)
    flags[:, 7::11] = 0
    k[:, :, 7::11], v[:, :, 7::11] = np.inf, np.nan
    Q, K, V = (to(T, t, "bf16")[0] for t in (q, k, v))
    kw = dict(kv_len=T.to_device(lens), kv_valid=T.to_device(flags))
    got = T.cross_attention(Q, K, V, **kw).numpy()
    count = (np.arange(n) < lens[:, None]) & (flags != 0)
    k2, v2 = (np.where(count[:, None, :, None], mxref.bf16_values(mxref.bf16_bits(t)), 0.0) for t in (k, v))
    want, size, big = crossref.attention(mxref.bf16_values(mxref.bf16_bits(q)), k2, v2, 0.125, count)
    assert (np.abs(got - want) - tolerance(want, size, big, d, n, "bf16", "f32", np.abs(v2).max())).max() <= 0
    v[1, 0, 40, 3] = np.nan                                    # (its flag is 0: 40 = 7 + 3 * 11)
    assert np.array_equal(T.cross_attention(Q, K, to(T, v, "bf16")[0], **kw).numpy(), got)
    v[1, 0, 41, 3] = np.nan
    got2 = T.cross_attention(Q, K, to(T, v, "bf16")[0], **kw).numpy()
    assert np.array_equal(got2[0], got[0]) and np.isnan(got2[1, :, 0, 3]).all()
    assert np.array_equal(np.delete(got2[1, :, 0], 3, 1), np.delete(got[1, :, 0], 3, 1))


@pytest.mark.parametrize("kv,size", [("bf16", 2.0 ** 8), ("bf16", 2.0 ** 20), ("bf16", 2.0 ** 55), ("f16", 2.0 ** 8), ("f16", 2.0 ** 14)])   # (f16 holds less than 2^16)
@pytest.mark.parametrize("rows,ranges", SHAPES)
def test_huge_logits(T, shape, rows, ranges, kv, size):  # noqa: F811
    """logits of 2^16 to 2^110 of either sign: all equal ones weigh the same (exactly: their products are powers of two), and where
    one stands above the others it takes all"""
    shape(rows, ranges)
    rng = np.random.default_rng(1)
    n, d = 300, 64
    v = rng.standard_normal((1, 1, n, d)).astype(np.float32)
    for sign in (1.0, -1.0):
        q = np.zeros((1, 1, 40, d), np.float32)
        q[..., 0] = size * 2.0 ** (np.arange(40) % 4 / 2 // 1)
        k = np.zeros((1, 1, n, d), np.float32)
        k[..., 0] = sign * size
        (Q, _), (K, _), (V, v2) = (to(T, t, kv) for t in (q, k, v))
        got = T.cross_attention(Q, K, V, scale=0.7).numpy()
        mean = v2[0, 0].astype(np.float64).mean(0)
        tol = (2 * U[kv] + 2 * (n + 64) * 2.0 ** -23) * np.abs(v2[0, 0]).mean(0) + 2.0 ** -24 * np.abs(mean)
        assert np.isfinite(got).all() and (np.abs(got[0, :, 0] - mean) <= tol).all()
        k[0, 0, 123, 0] *= 2.0 if sign > 0 else 0.5
        got = T.cross_attention(Q, to(T, k, kv)[0], V, scale=0.7).numpy()
        # one weight w: w v is exact (8 and 11 bits each), 1 / w and its product with w v round once each: 2 * 2^-24 of v
        assert (np.abs(got[0, :, 0] - v2[0, 0, 123]) <= 2.0 ** -23 * np.abs(v2[0, 0, 123])).all()


def test_flags_of_another_kind_are_refused(T):  # noqa: F811
    rng = np.random.default_rng(0)
    q, k = (to(T, rng.standard_normal((2, 1, n, 64)), "bf16")[0] for n in (3, 9))
    for flags in (np.ones((2, 9), np.float32), np.ones((2, 8), np.uint8), np.ones((1, 9), np.uint8)):
        with pytest.raises(ValueError):
            T.cross_attention(q, k, k, kv_valid=T.to_device(flags))
