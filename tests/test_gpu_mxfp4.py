"""MXFP4 on gfx950: quantization bit for bit, products against 64 bits.

Tolerances. Products of two E2M1 numbers are exact in fp32, products of an E2M1
number and a bf16 value too (2 + 8 bits); what is left is the fp32 sum of K
terms, at most one rounding (or truncation) per term: K 2^-23 sum |x w|, and
the output's own rounding, 2^-8 relative for bf16. Where every partial sum is a
multiple of a quarter below 2^22, sums are exact in any order and results must
be equal."""
import ctypes

import numpy as np
import pytest

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


def split(T, codes, byte):
    return T.SplitMXFP4(T.to_device(mxref.planes(codes, byte)), codes.shape[1], codes.shape[0])


def hard_rows(rng, rows, k):
    """values across the exponent range, with ties, zeros and non-finite blocks"""
    x = rng.standard_normal((rows, k)) * np.exp2(rng.integers(-20, 20, (rows, 1)))
    b = x.reshape(-1, 32)
    b[::3] = rng.integers(-32, 33, b[::3].shape) * 0.25        # ties of the scale 2^0 and its neighbours
    b[1::7] *= 2.0 ** -120                                     # (the scale stops at 2^-127)
    b[2::11] *= 2.0 ** 110
    with np.errstate(over="ignore"):                           # (some blocks become infinite)
        x = x.astype(np.float32)
    b = x.reshape(-1, 32)
    if len(b) > 8:
        b[3] = 0.0
        b[4] = -0.0
        b[5, 7] = np.inf
        b[6, 31] = -np.inf
        b[7, 0] = np.nan
        b[8] = np.float32(2.0 ** -149)
    return x


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 64), (3, 96), (77, 1024), (5, 2816), (1291, 160), (2, 8192), (4097, 32)])
def test_quantize_bits(T, rows, k, dtype):
    rng = np.random.default_rng(rows + k)
    x = hard_rows(rng, rows, k)
    if dtype == "bf16":
        x = mxref.bf16_values(mxref.bf16_bits(x))
    codes, byte = mxref.quantize(x)
    got_c, got_b = mxref.unplanes(T.mxfp4_quantize(dev(T, x, dtype)).buf.numpy(), rows, k)
    assert np.array_equal(got_b, byte) and np.array_equal(got_c, codes)
    blk = T.mxfp4_quantize(dev(T, x, dtype), split=False)
    assert np.array_equal(blk.numpy(), mxref.blocks(codes, byte))
    assert np.array_equal(T.mxfp4_repack(blk).buf.numpy(), mxref.planes(codes, byte))
    want = mxref.values(codes, byte).astype(np.float32)
    for q in (split(T, codes, byte), blk):
        for out in ("f32", "bf16"):
            got = host(T.mxfp4_dequantize(q, out))
            assert np.array_equal(got, want, equal_nan=True)
            assert np.array_equal(np.signbit(got) & ~np.isnan(got), np.signbit(want) & ~np.isnan(want))


def test_dequantize_every_code_and_scale(T):
    codes = np.tile(np.concatenate([np.arange(16), np.arange(16)[::-1]]).astype(np.uint8), (256, 1))
    byte = np.arange(256, dtype=np.uint8)[:, None]
    with np.errstate(over="ignore"):
        want = mxref.values(codes, byte).astype(np.float32)    # 2^128 and up: infinite
    for out in ("f32", "bf16"):
        assert np.array_equal(host(T.mxfp4_dequantize(split(T, codes, byte), out)), want, equal_nan=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_rows(T, dtype):
    """views: rows apart, 3-D with gaps, starts aligned to elements only; bytes behind the outputs stay"""
    rng = np.random.default_rng(5)
    full = rng.standard_normal((3, 9, 200)).astype(np.float32)
    if dtype == "bf16":
        full = mxref.bf16_values(mxref.bf16_bits(full))
    a = dev(T, full, dtype)
    for off, k in ((0, 64), (1, 96), (3, 192), (8, 160)):
        v = a.view(off + 200, (3, 7, k), (9 * 200, 200, 1))
        x = np.ascontiguousarray(full[:, 1:8, off:off + k].reshape(21, k))
        codes, byte = mxref.quantize(x)
        got = T.mxfp4_quantize(v).buf.numpy()
        assert np.array_equal(got, mxref.planes(codes, byte))
        out = dev(T, np.full_like(full, 7.0), dtype)
        ov = out.view(off + 200, (3, 7, k), (9 * 200, 200, 1))
        q = split(T, codes, byte)
        dq, dd = T.desc(q, T.MXFP4_SPLIT), T.desc(ov)
        dq.ne[1], dq.ne[2] = 7, 3
        T.check(T.load().tsk_mxfp4_dequantize(ctypes.byref(dq), ctypes.byref(dd), None))
        want = np.full_like(full, 7.0)
        want[:, 1:8, off:off + k] = mxref.values(codes, byte).reshape(3, 7, k)
        assert np.array_equal(host(out), want)
    # blocks with rows further apart than their bytes
    x = rng.standard_normal((5, 64)).astype(np.float32)
    codes, byte = mxref.quantize(x)
    buf = T.to_device(np.full((5, 50), 9, np.uint8))
    bv = buf.view(1, (5, 2, 17), (50, 17, 1))
    T.mxfp4_quantize(T.to_device(x), out=bv)
    got = buf.numpy()
    assert np.array_equal(got[:, 1:35].reshape(5, 2, 17), mxref.blocks(codes, byte))
    assert (got[:, 0] == 9).all() and (got[:, 35:] == 9).all()
    assert np.array_equal(T.mxfp4_repack(bv).buf.numpy(), mxref.planes(codes, byte))
    assert np.array_equal(host(T.mxfp4_dequantize(bv)), mxref.values(codes, byte).astype(np.float32))


def padded(T, rows, m, dtype):
    """an output of m columns in rows of 16-byte strides, all 3.0"""
    ld = (m + 7) // 8 * 8 + 8
    buf = dev(T, np.full((rows, ld), 3.0, np.float32), dtype)
    return buf, buf.view(0, (rows, m), (ld, 1))


def operands(rng, n, k, m, exact):
    wc, xc = rng.integers(0, 16, (m, k)).astype(np.uint8), rng.integers(0, 16, (n, k)).astype(np.uint8)
    lo, hi = (127, 129) if exact else (110, 135)
    wb, xb = (rng.integers(lo, hi, (r, k // 32)).astype(np.uint8) for r in (m, n))
    return wc, wb, xc, xb


SHAPES = [(1, 32, 16), (1, 64, 1), (1, 1024, 1000), (2, 96, 33), (3, 4096, 40), (8, 544, 65), (15, 128, 129), (16, 256, 64),
          (17, 160, 48), (33, 992, 100), (64, 2048, 256), (65, 288, 130), (77, 1024, 512), (129, 512, 257), (200, 1312, 384),
          (256, 256, 256), (257, 640, 300), (388, 1024, 1024), (511, 96, 511), (1100, 2816, 520)]


@pytest.mark.parametrize("n,k,m", SHAPES)
@pytest.mark.parametrize("act", ["mxfp4", "bf16", "f32"])
def test_products_equal_where_sums_are_exact(T, n, k, m, act):
    """codes times 1 or 2 (sums are multiples of a quarter, at most 2816 * 144 < 2^19): every result equal"""
    rng = np.random.default_rng(n * 31 + k + m)
    wc, wb, xc, xb = operands(rng, n, k, m, True)
    w = mxref.values(wc, wb)
    if act == "mxfp4":
        x, xd = mxref.values(xc, xb), split(T, xc, xb)
    else:
        x = rng.integers(-8, 9, (n, k)).astype(np.float32)
        xd = dev(T, x, act)
    want = x.astype(np.float64) @ w.T
    buf, y = padded(T, n, m, "f32")
    T.mul_mat(split(T, wc, wb), xd, out=y)
    got = buf.numpy()
    assert np.array_equal(got[:, :m], want.astype(np.float32))
    assert (got[:, m:] == 3.0).all()                           # nothing past the rows
    # the blocks are the planes' values; bias; bf16 output (the exact sums rounded once)
    bias = rng.integers(-64, 65, m).astype(np.float32)
    buf, y = padded(T, n, m, "bf16")
    T.mul_mat(T.to_device(mxref.blocks(wc, wb)), xd, bias=T.to_device(bias), out=y, a_type=T.MXFP4)
    got = host(buf)
    assert np.array_equal(got[:, :m], mxref.bf16_values(mxref.bf16_bits((want + bias).astype(np.float32))))
    assert (got[:, m:] == 3.0).all()


@pytest.fixture
def shape(T, monkeypatch):
    """force a launch shape of the products"""
    def force(cfg):
        monkeypatch.setenv("TSK_MX_CFG", str(cfg))
        T.init(0, reread=True)
    yield force
    monkeypatch.delenv("TSK_MX_CFG")
    T.init(0, reread=True)


@pytest.mark.parametrize("cfg", [1, 2, 3, 4, 5, 6, 7, 8, 9, 11, 12, 13, 14, 15])
@pytest.mark.parametrize("act", ["mxfp4", "bf16", "f32"])
def test_every_launch_shape(T, shape, cfg, act):
    """ragged in rows, outputs and K (blocks of scales whole, by twos and odd; K shorter than a stage and longer than a
    chunk of scales), equal to the exact sums; a NaN scale right behind the end of a row reaches only its own"""
    shape(cfg)
    rng = np.random.default_rng(cfg)
    for n, k, m in ((300, 1152, 273), (257, 2176, 260), (131, 192, 130), (70, 1088, 515), (270, 160, 300), (33, 32, 65), (19, 96, 17),
                    (140, 2592, 150)):
        wc, wb, xc, xb = operands(rng, n, k, m, True)
        wb[m // 2, 0] = 255
        if act == "mxfp4":
            xb[n // 2, 0] = 255
            x, xd = mxref.values(xc, xb), split(T, xc, xb)
        else:
            x = rng.integers(-8, 9, (n, k)).astype(np.float32)
            xd = dev(T, x, act)
        want = (x.astype(np.float64) @ mxref.values(wc, wb).T).astype(np.float32)
        buf, y = padded(T, n, m, "f32")
        T.mul_mat(split(T, wc, wb), xd, out=y)
        got = buf.numpy()
        assert np.array_equal(got[:, :m], want, equal_nan=True), (n, k, m)
        assert np.isnan(want).sum() == n + ((m - 1) if act == "mxfp4" else 0)
        assert (got[:, m:] == 3.0).all()


@pytest.mark.parametrize("n,k,m", [(1, 8192, 96), (4, 1024, 2048), (30, 4096, 200), (200, 1536, 1000), (1025, 2048, 640)])
@pytest.mark.parametrize("act", ["mxfp4", "bf16", "f32"])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_products_of_real_values(T, n, k, m, act, out):
    rng = np.random.default_rng(n + k + m)
    x = rng.standard_normal((n, k)).astype(np.float32) * np.exp2(rng.integers(-3, 4, (n, 1))).astype(np.float32)
    wc, wb = mxref.quantize(rng.standard_normal((m, k)).astype(np.float32) * np.float32(k ** -0.5))
    bias = rng.standard_normal(m).astype(np.float32)
    if act == "mxfp4":
        xc, xb = mxref.quantize(x)
        xv, xd = mxref.values(xc, xb), T.mxfp4_quantize(T.to_device(x))
    else:
        xv, xd = mxref.bf16_values(mxref.bf16_bits(x)).astype(np.float64), dev(T, x, act)   # f32 is rounded to bf16
    w = mxref.values(wc, wb)
    want = xv @ w.T + bias
    size = np.abs(xv) @ np.abs(w).T + np.abs(bias)
    got = host(T.mul_mat(split(T, wc, wb), xd, bias=T.to_device(bias), out_dtype=out)).astype(np.float64)
    tol = (k + 1) * 2.0 ** -23 * size + (2.0 ** -8 * np.abs(want) if out == "bf16" else 0.0)
    assert (np.abs(got - want) <= tol).all()
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel <= (2.0 ** -8 if out == "bf16" else 1e-6)


@pytest.mark.parametrize("act", ["mxfp4", "bf16", "f32"])
@pytest.mark.parametrize("n", [2, 40, 300])
def test_rows_of_their_own(T, act, n):
    """a NaN scale or an infinite activation touches its own row or column alone, and every row is the same
    whatever rows stand beside it in a call of the same size"""
    rng = np.random.default_rng(n)
    k, m = 256, 160
    wc, wb, xc, xb = operands(rng, n, k, m, True)
    wb[5, 3] = 255
    x = rng.integers(-8, 9, (n, k)).astype(np.float32)
    if act == "mxfp4":
        xb[1, 2] = 255
        x, xd = mxref.values(xc, xb), split(T, xc, xb)
    else:
        x[1, 70] = np.inf
        xd = dev(T, x, act)
    y = T.mul_mat(split(T, wc, wb), xd).numpy()
    w = mxref.values(wc, wb)
    rows, cols = np.arange(n) != 1, np.arange(m) != 5
    assert np.isnan(y[:, 5]).all()
    assert not np.isfinite(y[1]).any() or act != "mxfp4"
    assert np.isnan(y[1]).all() if act == "mxfp4" else not np.isfinite(y[1][w[:, 70] != 0]).any()
    assert np.array_equal(y[rows][:, cols], (x[rows].astype(np.float64) @ w[cols].T).astype(np.float32))


def test_batched_and_strided_activations(T):
    """b with outer extents: uniform rows in one product, gaps slice by slice; planes over all rows"""
    rng = np.random.default_rng(3)
    k, m = 192, 72
    wc, wb, _, _ = operands(rng, 1, k, m, True)
    w, W = mxref.values(wc, wb), split(T, wc, wb)
    x = rng.integers(-8, 9, (2, 3, 50, 200)).astype(np.float32)
    xd = T.to_device(x)
    v = xd.view(8, (2, 3, 40, k), (3 * 50 * 200, 50 * 200, 200, 1))
    want = (x[:, :, :40, 8:8 + k].astype(np.float64) @ w.T).astype(np.float32)
    assert np.array_equal(T.mul_mat(W, v).numpy(), want)
    # planes of (2, 3, 40) rows into an output with gaps between the slices
    xc, xb = mxref.quantize(x[:, :, :40, :k].reshape(-1, k))
    q = split(T, xc, xb)
    out = T.to_device(np.full((2, 3, 44, m), 5.0, np.float32))
    dq, dw, dd = T.desc(q, T.MXFP4_SPLIT), T.desc(W, T.MXFP4_SPLIT), T.desc(out.view(0, (2, 3, 40, m), out.strides))
    dq.ne[1], dq.ne[2], dq.ne[3] = 40, 3, 2
    T.check(T.load().tsk_mul_mat(ctypes.byref(dw), ctypes.byref(dq), None, ctypes.byref(dd), None))
    got = out.numpy()
    assert np.array_equal(got[:, :, :40], (mxref.values(xc, xb) @ w.T).astype(np.float32).reshape(2, 3, 40, m))
    assert (got[:, :, 40:] == 5.0).all()


@pytest.mark.parametrize("act", ["mxfp4", "bf16", "f32"])
@pytest.mark.parametrize("n,k,m", [(1, 2048, 512), (60, 4096, 96), (300, 1024, 512), (96, 8192, 64)])
def test_bits_of_every_call(T, act, n, k, m):
    """the same bits eager, on another stream, without allocation and replayed from a graph between eager work"""
    rng = np.random.default_rng(k)
    W = T.mxfp4_quantize(T.to_device(rng.standard_normal((m, k)).astype(np.float32)))
    xs = [rng.standard_normal((n, k)).astype(np.float32) for _ in range(3)]
    mk = (lambda x: T.mxfp4_quantize(T.to_device(x))) if act == "mxfp4" else (lambda x: dev(T, x, act))
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
    buf = x.buf if act == "mxfp4" else x
    for i in (1, 2, 0, 1):
        src = mk(xs[i])
        T._hipcheck(T.hip().hipMemcpy(ctypes.c_void_p(buf.ptr), ctypes.c_void_p((src.buf if act == "mxfp4" else src).ptr),
                                      buf.nbytes, 3), "hipMemcpy D2D")
        T.mul_mat(W, mk(xs[0]))                                # eager work on another stream between the replays
        T.synchronize()
        g.launch()
        st.synchronize()
        assert np.array_equal(out.numpy(), want[i])
    g.destroy()
    st.destroy()
