"""8-bit rows with one scale each on gfx950: quantization bit for bit, products against exact sums.

Tolerances. Integer sums are exact. What follows them is rounded in fp32: the sum itself, times the token's scale, times
the channel's, plus bias: three roundings of the product, 3 * 2^-24 of it (3.1 with their products), and one of the result;
bf16 outputs are off by 2^-8 of theirs more."""
import ctypes

import numpy as np
import pytest

import crossref
import mxref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    from __graft_entry__ import ensure_built, load_tsk
    ensure_built()
    t = load_tsk()
    t.init(0)
    return t


def dev(T, x, dtype="f32"):
    return T.to_device(x) if dtype == "f32" else T.bf16_to_device(mxref.bf16_bits(x))


def host(a):
    return mxref.bf16_values(a.numpy()) if a.dtype == "bf16" else a.numpy()


def typed(x, dtype):
    return mxref.bf16_values(mxref.bf16_bits(x)) if dtype == "bf16" else x


def planes(T, q, d):
    return T.SplitI8(T.to_device(crossref.i8_planes(q, d)), q.shape[1], q.shape[0])


def check_planes(sp, x, k):
    rows = x.size // k
    q, d = crossref.i8_quantize(x.reshape(rows, k))
    got, s = crossref.i8_unplanes(sp.buf.numpy(), rows, k)
    assert np.array_equal(s.view(np.uint32)[~np.isnan(d)], d.view(np.uint32)[~np.isnan(d)]) and np.isnan(s[np.isnan(d)]).all()
    assert np.array_equal(got[:, :k], q) and not got[:, k:].any()


def hard_rows(rng, rows, k):
    """values across the exponent range, with ties, zeros and what is not finite"""
    x = rng.standard_normal((rows, k)) * np.exp2(rng.integers(-30, 30, (rows, 1)))
    x[::4] = rng.integers(-254, 255, x[::4].shape) * 0.5       # ties of the scale 1 and its neighbours
    x[::4, 0] = 127.0
    x[1::8] = rng.integers(-254, 255, x[1::8].shape) * 1.5     # of the scale 3
    x[1::8, 0] = 381.0
    x = x.astype(np.float32)
    if rows > 12:
        x[2], x[3], x[5] = 0.0, -0.0, np.float32(2.0 ** -149)
        x[6] = np.float32(3e38) * np.sign(rng.standard_normal(k)).astype(np.float32)
        x[7, k // 2], x[10, k - 1], x[11, 0] = np.inf, -np.inf, np.nan
        x[12] *= np.float32(2.0 ** -90)
    return x


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 5), (3, 16), (40, 17), (40, 127), (65, 129), (33, 1000), (40, 1024), (21, 2816),
                                    (17, 4104), (19, 8200), (5, 16384), (16, 16390)])
def test_quantize_bits(T, dtype, rows, k):
    x = typed(hard_rows(np.random.default_rng(k), rows, k), dtype)
    sp = T.i8_quantize(dev(T, x, dtype))
    check_planes(sp, x, k)
    q, d = crossref.i8_quantize(x)
    v = q.astype(np.float32) * d[:, None]
    assert np.array_equal(T.i8_dequantize(sp).numpy(), v, equal_nan=True)
    assert np.array_equal(host(T.i8_dequantize(sp, "bf16")), typed(v, "bf16"), equal_nan=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_rows(T, dtype):
    """rows of a 4-D view off 16 bytes, broadcast ones, and back into another"""
    rng = np.random.default_rng(4)
    x = typed(rng.standard_normal((2, 3, 5, 61)).astype(np.float32), dtype)
    xd = dev(T, x, dtype)
    v = xd.view(1, (2, 3, 4, 50), xd.strides)
    want = np.ascontiguousarray(x[:, :, :4, 1:51])
    sp = T.i8_quantize(v)
    check_planes(sp, want, 50)
    out = dev(T, np.full((2, 4, 3, 53), 7.0, np.float32), dtype)
    T.i8_dequantize(sp, out=out.view(3, (2, 3, 4, 50), (4 * 3 * 53, 53, 3 * 53, 1)))
    q, d = crossref.i8_quantize(want.reshape(-1, 50))
    got = host(out)
    y = typed((q.astype(np.float32) * d[:, None]).reshape(2, 3, 4, 50), dtype)
    assert np.array_equal(got[..., 3:].transpose(0, 2, 1, 3), y) and (got[..., :3] == 7.0).all()
    same = T.i8_quantize(xd.view(0, (4, 61), (0, 1)))
    check_planes(same, np.broadcast_to(x[0, 0, 0], (4, 61)), 61)


def want_linear(x, w, bias, dtype):
    """x, w: (integers, scales): the result, and how far it may be off"""
    acc = (x[0].astype(np.int64) @ w[0].astype(np.int64).T).astype(np.float64)
    prod = acc * x[1].astype(np.float64)[:, None] * w[1].astype(np.float64)[None]
    y = prod + (0 if bias is None else bias.astype(np.float64))
    return y, 3.1 * 2.0 ** -24 * np.abs(prod) + (2.0 ** -24 + (2.0 ** -8 if dtype == "bf16" else 0)) * (np.abs(y) + np.abs(prod) * 2.0 ** -22)


def off(got, want, tol):
    return float((np.abs(got.astype(np.float64) - want) - tol).max())


SIZES = [(1, 16, 16), (1, 1, 1), (1, 1024, 6144), (2, 100, 130), (8, 8192, 96), (16, 333, 64), (17, 64, 256), (33, 2816, 70),
         (77, 1024, 1024), (130, 1000, 260), (388, 1024, 512), (300, 48, 2050), (513, 4096, 192), (1292, 160, 1024), (1000, 2047, 515)]


@pytest.mark.parametrize("act", ["i8", "f32", "bf16"])
@pytest.mark.parametrize("n,k,m", SIZES)
def test_linear(T, act, n, k, m):
    rng = np.random.default_rng(n * 7 + k)
    x = typed((rng.standard_normal((n, k)) * np.exp(rng.standard_normal((n, 1)))).astype(np.float32), act)
    w = crossref.i8_quantize((rng.standard_normal((m, k)) * np.exp(rng.standard_normal((m, 1)))).astype(np.float32))
    bias = (rng.standard_normal(m) * 3).astype(np.float32)
    xq, W = crossref.i8_quantize(x), planes(T, *w)
    per = 8 if act == "bf16" else 4
    if act == "i8":
        X = planes(T, *xq)
    else:                                                      # rows on 16-byte starts
        pad = np.full((n, (k + per - 1) // per * per), 1e30, np.float32)
        pad[:, :k] = x
        P = dev(T, pad, act)
        X = P.view(0, (n, k), P.strides)
    for b, dtype in ((None, "f32"), (bias, "f32"), (bias, "bf16")):
        ldy = (m + 7) // 8 * 8
        out = dev(T, np.full((n, ldy), 9.0, np.float32), dtype)
        T.mul_mat(W, X, bias=None if b is None else T.to_device(b), out=out.view(0, (n, m), out.strides))
        got = host(out)
        y, tol = want_linear(xq, w, b, dtype)
        assert off(got[:, :m], y, tol) <= 0, (b is None, dtype)
        assert (got[:, m:] == 9.0).all()


@pytest.mark.parametrize("n", [1, 3, 16, 40, 300])
@pytest.mark.parametrize("k", [131071, 130000])
def test_largest_sums(T, n, k):
    """-128 throughout, longest rows: sums of almost 2^31, which fp32 rounds once"""
    m = 37
    q = lambda r: (np.full((r, k), -128, np.int8), np.ones(r, np.float32))
    y = T.mul_mat(planes(T, *q(m)), planes(T, *q(n)), out=None if m % 4 == 0 else T.empty((n, 40)).view(0, (n, m), (40, 1)))
    out = np.empty((n, 40), np.float32)
    T.synchronize()
    T._hipcheck(T.hip().hipMemcpy(ctypes.c_void_p(out.ctypes.data), ctypes.c_void_p(y.ptr), out.nbytes - 12, 2), "hipMemcpy D2H")
    assert (out[:, :m] == np.float32(16384.0 * k)).all()


@pytest.mark.parametrize("n", [2, 50, 400])
def test_scales_that_are_not_finite(T, n):
    """a token's or a channel's: its row or column, nothing else"""
    rng = np.random.default_rng(n)
    k, m = 200, 96
    x, w = (crossref.i8_quantize(rng.standard_normal((r, k)).astype(np.float32)) for r in (n, m))
    x[1][1], w[1][5], w[1][7] = np.nan, np.nan, np.inf
    y = T.mul_mat(planes(T, *w), planes(T, *x)).numpy()
    assert np.isnan(y[1]).all() and np.isnan(y[:, 5]).all() and not np.isfinite(y[:, 7]).any()
    rows, cols = np.arange(n) != 1, ~np.isin(np.arange(m), (5, 7))
    want, tol = want_linear((x[0][rows], x[1][rows]), (w[0][cols], w[1][cols]), None, "f32")
    assert off(y[rows][:, cols], want, tol) <= 0


def test_batched_and_strided_activations(T):
    """b with outer extents and gaps, dst with gaps between the slices, planes over all rows"""
    rng = np.random.default_rng(3)
    k, m = 200, 72
    w = crossref.i8_quantize(rng.standard_normal((m, k)).astype(np.float32))
    W = planes(T, *w)
    x = rng.standard_normal((2, 3, 50, 208)).astype(np.float32)
    xd = T.to_device(x)
    v = xd.view(8, (2, 3, 40, k), xd.strides)
    xq = crossref.i8_quantize(np.ascontiguousarray(x[:, :, :40, 8:]).reshape(-1, k))
    want, tol = want_linear(xq, w, None, "f32")
    assert off(T.mul_mat(W, v).numpy().reshape(-1, m), want, tol) <= 0
    out = T.to_device(np.full((2, 3, 44, m), 5.0, np.float32))
    T.mul_mat(W, v, out=out.view(0, (2, 3, 40, m), out.strides))
    got = out.numpy()
    assert off(got[:, :, :40].reshape(-1, m), want, tol) <= 0 and (got[:, :, 40:] == 5.0).all()
    X, out = planes(T, *xq), T.to_device(np.full((2, 3, 44, m), 5.0, np.float32))
    dq, dw, dd = T.desc(X, T.I8_SPLIT), T.desc(W, T.I8_SPLIT), T.desc(out.view(0, (2, 3, 40, m), out.strides))
    dq.ne[1], dq.ne[2], dq.ne[3] = 40, 3, 2
    T.check(T.load().tsk_mul_mat(ctypes.byref(dw), ctypes.byref(dq), None, ctypes.byref(dd), None))
    got = out.numpy()
    assert off(got[:, :, :40].reshape(-1, m), want, tol) <= 0 and (got[:, :, 40:] == 5.0).all()


@pytest.mark.parametrize("act", ["i8", "bf16", "f32"])
@pytest.mark.parametrize("n,k,m", [(1, 2048, 512), (60, 4096, 96), (300, 1024, 512), (96, 8192, 64), (5, 520, 1000)])
def test_bits_of_every_call(T, act, n, k, m):
    """the same bits eager, on another stream, without allocation and replayed from a graph between eager work"""
    rng = np.random.default_rng(k)
    W = T.i8_quantize(T.to_device(rng.standard_normal((m, k)).astype(np.float32)))
    xs = [rng.standard_normal((n, k)).astype(np.float32) for _ in range(3)]
    mk = (lambda x: T.i8_quantize(T.to_device(x))) if act == "i8" else (lambda x: dev(T, x, act))
    want = [T.mul_mat(W, mk(x)).numpy() for x in xs]
    assert np.array_equal(T.mul_mat_noalloc(W, mk(xs[0])).numpy(), want[0])
    st = T.Stream()
    x = mk(xs[0])
    out = T.to_device(np.zeros((n, m), np.float32))
    T.synchronize()
    T.mul_mat(W, x, out=out, stream=st)                        # (its workspace, if any, exists before the capture)
    st.synchronize()
    assert np.array_equal(out.numpy(), want[0])
    g = T.Graph(st, lambda: T.mul_mat(W, x, out=out, stream=st))
    buf = x.buf if act == "i8" else x
    for i in (1, 2, 0, 1):
        src = mk(xs[i])
        T._hipcheck(T.hip().hipMemcpy(ctypes.c_void_p(buf.ptr), ctypes.c_void_p((src.buf if act == "i8" else src).ptr),
                                      buf.nbytes, 3), "hipMemcpy D2D")
        T.mul_mat(W, mk(xs[0]))                                # eager work on another stream between the replays
        T.synchronize()
        g.launch()
        st.synchronize()
        assert np.array_equal(out.numpy(), want[i])
    g.destroy()
    st.destroy()


@pytest.mark.parametrize("n", [1, 8, 20, 77, 400])
def test_rows_do_not_depend_on_the_batch(T, n):
    """a row's bits are those that it has alone: sums are exact whatever the tile"""
    rng = np.random.default_rng(n)
    W = T.i8_quantize(T.to_device(rng.standard_normal((300, 1000)).astype(np.float32)))
    x = rng.standard_normal((n, 1000)).astype(np.float32)
    y = T.mul_mat(W, T.to_device(x)).numpy()
    for i in (0, n // 2, n - 1):
        assert np.array_equal(T.mul_mat(W, T.to_device(x[i:i + 1])).numpy()[0], y[i])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 7), (5, 40), (14, 64), (9, 100), (388, 1024), (33, 1000), (4, 4096), (2, 9000), (3, 20000),
                                    (2, 20001)])
def test_block_norm_into_8_bit_rows(T, dtype, rows, c):
    """the integers of the f32 output of the same call"""
    rng = np.random.default_rng(c)
    x = dev(T, rng.standard_normal((rows, c)).astype(np.float32) * 3 + 0.5, dtype)
    scale, shift = (T.to_device(rng.standard_normal(c).astype(np.float32)) for _ in range(2))
    for kw in ({"pre": T.NORM_LAYER, "scale": scale, "shift": shift}, {"pre": T.NORM_RMS, "pre_w": scale}, {"pre": T.NORM_NONE}):
        y = T.to_device(np.zeros((rows, c), np.float32))
        sp = T.SplitI8(T.to_device(np.full(rows * ((c + 15) // 16 * 16 + 4), 99, np.uint8)), c, rows)
        T.block_norm(x, dst=y, **kw)
        T.block_norm(x, dst=sp, **kw)
        check_planes(sp, y.numpy(), c)


def test_block_norm_of_rows_that_are_not_finite(T):
    x = np.random.default_rng(1).standard_normal((6, 96)).astype(np.float32)
    x[1, 3], x[4, 95] = np.inf, np.nan
    x[2] = 0
    sp = T.SplitI8(T.to_device(np.full(6 * 100, 99, np.uint8)), 96, 6)
    T.block_norm(T.to_device(x), pre=T.NORM_NONE, dst=sp)
    check_planes(sp, x, 96)


@pytest.mark.parametrize("cfg", [1, 2, 3, 4, 5, 6, 7, 8, 11, 12, 13])
def test_each_shape(T, monkeypatch, cfg):
    """every kernel's tiles over ragged rows, outputs and depths; what lies behind the outputs stays"""
    rng = np.random.default_rng(cfg)
    monkeypatch.setenv("TSK_I8_CFG", str(cfg))
    T.init(0, reread=True)
    try:
        for n, k, m in ((5, 33, 20), (300, 1000, 515), (1, 1, 1), (270, 64, 258), (257, 129, 1), (33, 4100, 300), (1, 300, 260)):
            x = crossref.i8_quantize((rng.standard_normal((n, k)) * np.exp(rng.standard_normal((n, 1)))).astype(np.float32))
            w = crossref.i8_quantize(rng.standard_normal((m, k)).astype(np.float32))
            bias = rng.standard_normal(m).astype(np.float32)
            for b, dtype in ((None, "bf16"), (bias, "f32")):
                ldy = (m + 7) // 8 * 8
                out = dev(T, np.full((n, ldy), 9.0, np.float32), dtype)
                T.mul_mat(planes(T, *w), planes(T, *x), bias=None if b is None else T.to_device(b), out=out.view(0, (n, m), out.strides))
                got = host(out)
                y, tol = want_linear(x, w, b, dtype)
                assert off(got[:, :m], y, tol) <= 0, (n, k, m, dtype)
                assert (got[:, m:] == 9.0).all()
    finally:
        monkeypatch.delenv("TSK_I8_CFG")
        T.init(0, reread=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("amax", [127.0, 254.0, 1.0, 127.0 * 2.0 ** -90, 126.99999])
def test_codes_next_to_a_half(T, dtype, amax):
    """every half between two integers, exact and one step of the type to either side, in rows of a known scale"""
    d = np.float32(amax) / np.float32(127.0)
    halves = (np.arange(-127, 127) + 0.5).astype(np.float64) * np.float64(d)
    x = typed(halves.astype(np.float32), dtype)
    if dtype == "f32":
        near = [x, np.nextafter(x, np.float32(np.inf)), np.nextafter(x, np.float32(-np.inf))]
    else:
        step = np.abs(x) * np.float32(2.0 ** -7)
        near = [x, typed(x + step, dtype), typed(x - step, dtype)]
    rows = np.stack([np.concatenate([[np.float32(amax)], np.clip(t, -np.float32(amax), np.float32(amax))]).astype(np.float32) for t in near])
    rows = typed(rows, dtype)
    check_planes(T.i8_quantize(dev(T, rows, dtype)), rows, rows.shape[1])


def test_two_streams(T):
    """products on two streams keep their quantized activations apart"""
    rng = np.random.default_rng(2)
    W = T.i8_quantize(T.to_device(rng.standard_normal((260, 1030)).astype(np.float32)))
    xs = [T.to_device(rng.standard_normal((n, 1032)).astype(np.float32)).view(0, (n, 1030), (1032, 1)) for n in (90, 400)]
    want = [T.mul_mat(W, x).numpy() for x in xs]
    st, outs = [T.Stream(), T.Stream()], [T.empty(w.shape) for w in want]
    T.synchronize()
    for _ in range(20):
        for s, x, o in zip(st, xs, outs):
            T.mul_mat(W, x, out=o, stream=s)
    for s in st:
        s.synchronize()
    for o, w in zip(outs, want):
        assert np.array_equal(o.numpy(), w)
    for s in st:
        s.destroy()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k", [(70, 40), (30, 500), (20, 1500), (9, 2048), (15, 6001), (300, 8185), (300, 8192), (5, 8000), (1030, 24)])
def test_rows_of_each_width(T, dtype, rows, k):
    """rows of every number of threads, few and many, on 16 bytes and not"""
    x = typed(hard_rows(np.random.default_rng(rows + k), rows, k), dtype)
    for first in (0, 1):                                       # (1: every row starts off 16 bytes)
        ld = (k + 7) // 8 * 8 + 8
        pad = np.full((rows, ld), 1e30, np.float32)
        pad[:, first:first + k] = x
        P = dev(T, pad, dtype)
        sp = T.i8_quantize(P.view(first, (rows, k), P.strides))
        check_planes(sp, x, k)
        q, d = crossref.i8_quantize(x)
        out = dev(T, np.full((rows, ld), 7.0, np.float32), dtype)
        T.i8_dequantize(sp, out=out.view(first, (rows, k), out.strides))
        got = host(out)
        assert np.array_equal(got[:, first:first + k], typed(q.astype(np.float32) * d[:, None], dtype), equal_nan=True)
        assert (got[:, :first] == 7.0).all() and (got[:, first + k:] == 7.0).all()
