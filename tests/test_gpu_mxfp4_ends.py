"""MXFP4 and the block norm where calls are rare: strides of extents of 1, broadcast rows, starts off 16 bytes, offsets
past 32 bits, other streams, graphs, bound workspaces. Inputs are small integers where sums are then exact, so results
are equal; the norm's bounds are those of its own tests (u = 2^-24 an operation, 2^-8 for a bf16 result)."""
import ctypes

import numpy as np
import pytest

import mxref
from test_gpu_block_norm import make, norm_and_bound, U
from test_gpu_mxfp4 import T, dev, host, operands, split  # noqa: F401  (T: fixture)

pytestmark = pytest.mark.gpu


def copy(T, dst, offset, a):
    """host array a to byte `offset` of dst"""
    a = np.ascontiguousarray(a)
    T._hipcheck(T.hip().hipMemcpy(ctypes.c_void_p(dst.ptr + offset), ctypes.c_void_p(a.ctypes.data), a.nbytes, 1), "hipMemcpy H2D")


def fetch(T, src, offset, shape, dtype):
    out = np.empty(shape, dtype)
    T.synchronize()
    T._hipcheck(T.hip().hipMemcpy(ctypes.c_void_p(out.ctypes.data), ctypes.c_void_p(src.ptr + offset), out.nbytes, 2), "hipMemcpy D2H")
    return out


def test_planes_of_other_sizes(T):
    """planes too small for their rows, or of other rows than x's, never reach a kernel"""
    x = T.to_device(np.ones((8, 64), np.float32))
    with pytest.raises(ValueError):
        T.SplitMXFP4(T.empty((4 * 34 - 1,), "u8"), 64, 4)
    four = T.SplitMXFP4(T.empty((4 * 34,), "u8"), 64, 4)
    with pytest.raises(ValueError):
        T.mxfp4_quantize(x, out=four)
    with pytest.raises(ValueError):
        T.block_norm(x, dst=four)


def test_strides_of_extents_of_one(T):
    """the stride of an extent of 1 is never a row's distance"""
    rng = np.random.default_rng(1)
    k, m = 96, 40
    wc, wb, _, _ = operands(rng, 1, k, m, True)
    w, W = mxref.values(wc, wb), split(T, wc, wb)
    x = rng.integers(-8, 9, (5, 200)).astype(np.float32)
    xd = T.to_device(x)
    want = (x[:, :k].astype(np.float64) @ w.T).astype(np.float32)
    for shape, st in (((5, 1, 1, k), (200, 8, 16, 1)), ((1, 5, 1, k), (8, 200, 4, 1)), ((1, 1, 5, k), (12, 4, 200, 1))):
        out = T.to_device(np.full((5, 64), 7.0, np.float32))
        ov = out.view(0, shape[:3] + (m,), tuple(64 if s == 200 else 4 for s in st[:3]) + (1,))
        T.mul_mat(W, xd.view(0, shape, st), out=ov)
        got = out.numpy()
        assert np.array_equal(got[:, :m], want) and (got[:, m:] == 7.0).all()
    # five rows as (5, 1, 1) blocks whose inner strides say nothing
    q = x[:, :k]
    codes, byte = mxref.quantize(q)
    buf = T.to_device(np.full((5, 64), 9, np.uint8))
    dx, db = T.desc(xd.view(0, (5, 1, 1, k), (200, 4, 4, 1))), T.desc(buf.view(0, (5, 3, 17), (64, 17, 1)), T.MXFP4)
    db.ne[1], db.ne[2], db.ne[3] = 1, 1, 5
    db.nb[1], db.nb[2], db.nb[3] = 3, 5, 64
    T.check(T.load().tsk_mxfp4_quantize(ctypes.byref(dx), ctypes.byref(db), None))
    got = buf.numpy()
    assert np.array_equal(got[:, :51].reshape(5, 3, 17), mxref.blocks(codes, byte)) and (got[:, 51:] == 9).all()
    y = T.to_device(np.zeros((5, k), np.float32))
    dy = T.desc(y.view(0, (5, 1, 1, k), (k, 4, 4, 1)))
    T.check(T.load().tsk_mxfp4_dequantize(ctypes.byref(db), ctypes.byref(dy), None))
    assert np.array_equal(y.numpy(), mxref.values(codes, byte).astype(np.float32))


@pytest.mark.parametrize("n", [3, 40, 200])
@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_broadcast_rows(T, n, act):
    """activations of stride 0: the same row n times"""
    rng = np.random.default_rng(n)
    k, m = 288, 300
    wc, wb, _, _ = operands(rng, 1, k, m, True)
    x = rng.integers(-8, 9, (1, k)).astype(np.float32)
    v = dev(T, x, act).view(0, (n, k), (0, 1))
    want = (x.astype(np.float64) @ mxref.values(wc, wb).T).astype(np.float32)
    assert np.array_equal(T.mul_mat(split(T, wc, wb), v).numpy(), np.repeat(want, n, 0))
    q = T.mxfp4_quantize(v)
    codes, byte = mxref.quantize(np.repeat(x, n, 0))
    assert np.array_equal(q.buf.numpy(), mxref.planes(codes, byte))


@pytest.mark.parametrize("c", [96, 1024, 8224, 20000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_into_4_bits_from_any_start(T, c, dtype):
    """rows that start off 16 bytes, the residual in place: the residual and the codes of what is within the norm's
    bounds of the 64-bit one"""
    rng = np.random.default_rng(c)
    d = make(rng, (2, 3, c), dtype, "batch", True, True)
    wide = np.zeros((2, 3, c + 7), np.float32)
    wide[:, :, 1:1 + c] = d["x"]
    keep = {k: T.to_device(d[k]) for k in ("gate", "post_w", "pre_w", "scale", "shift")}
    a, y = dev(T, wide, dtype), dev(T, d["y"], dtype)
    x = a.view(1, (2, 3, c), (3 * (c + 7), c + 7, 1))
    q = T.SplitMXFP4(T.empty((6 * c // 32 * 17,), "u8"), c, 6)
    T.block_norm(x, y, gate=keep["gate"], post=T.NORM_LAYER, post_w=keep["post_w"], pre=T.NORM_RMS, pre_w=keep["pre_w"],
                 scale=keep["scale"], shift=keep["shift"], res=x, dst=q)
    got = host(a).astype(np.float64)
    assert (got[:, :, 0] == 0).all() and (got[:, :, 1 + c:] == 0).all()
    r = got[:, :, 1:1 + c]
    e = {k: v.astype(np.float64) for k, v in d.items()}
    b, bb = norm_and_bound(e["y"], 1, 1e-5, e["post_w"])
    want = e["x"] + e["gate"] * b
    bound = 3 * U * np.abs(e["x"]) + np.abs(e["gate"]) * (bb + 3 * U * np.abs(b)) + (2.0 ** -8 * np.abs(want) if dtype == "bf16" else 0)
    assert (np.abs(r - want) <= bound).all()
    h, bh = norm_and_bound(r, 2, 1e-5, e["pre_w"])
    bh = bh * np.abs(1 + e["scale"]) + 3 * U * np.abs(h) * (1 + np.abs(e["scale"]))
    h = h * (1 + e["scale"]) + e["shift"]
    h, bh = (v.reshape(6, c // 32, 32) for v in (h, bh + 2 * U * np.abs(h)))
    codes, byte = mxref.unplanes(q.buf.numpy(), 6, c)
    scale = 2.0 ** (byte.astype(np.float64) - 127)[..., None]
    amax, slack = np.abs(h).max(-1, keepdims=True), bh.max(-1, keepdims=True)
    assert (amax >= 4 * scale - slack).all() and (amax < 8 * scale + slack).all()
    v = mxref.values(codes, byte).reshape(h.shape) / scale
    half = np.select([np.abs(v) < 2, np.abs(v) < 4], [0.25, 0.5], 1.0)      # half the wider step beside a code
    assert (np.abs(v - np.clip(h / scale, -6, 6)) <= half + bh / scale).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_offsets_past_32_bits_in_rows(T, dtype):
    """520 rows 8 MiB apart: activations, outputs, the norm and the quantizer past 4 GiB"""
    rng = np.random.default_rng(4)
    n, k, m, ld, es = 520, 64, 512, 1 << 23, 4 if dtype == "f32" else 2
    wc, wb, _, _ = operands(rng, 1, k, m, True)
    x = rng.integers(-8, 9, (n, k)).astype(np.float32)
    a, o = T.empty(((n - 1) * ld + 65536,), "u8"), T.empty(((n - 1) * ld + 65536,), "u8")
    bits = x if dtype == "f32" else mxref.bf16_bits(x).astype(np.uint16)
    for i in range(n):
        copy(T, a, i * ld, bits[i])
    rows = lambda base, at, cols, dt: T.DeviceArray((n, cols), dt, _base=base, _ptr=base.ptr + at, _strides=(ld // (2 if dt == "bf16" else 4), 1))
    last = [0, 1, 255, 256, 511, 512, 513, n - 1]
    read = lambda at, cols: np.stack([fetch(T, o, i * ld + at, (cols,), np.float32) for i in last])
    xv, zv = rows(a, 0, k, dtype), rows(o, 8192, k, "f32")
    T.mul_mat(split(T, wc, wb), xv, out=rows(o, 0, m, "f32"))
    assert np.array_equal(read(0, m), (x.astype(np.float64) @ mxref.values(wc, wb).T).astype(np.float32)[last])
    codes, byte = mxref.quantize(x)
    assert np.array_equal(T.mxfp4_quantize(xv).buf.numpy(), mxref.planes(codes, byte))
    T.mxfp4_dequantize(split(T, codes, byte), out=zv)
    assert np.array_equal(read(8192, k), mxref.values(codes, byte)[last].astype(np.float32))
    rv = rows(o, 16384, k, dtype)
    T.block_norm(xv, xv, pre=T.NORM_LAYER, res=rv, dst=zv)
    r = np.stack([fetch(T, o, i * ld + 16384, (k,), np.float32 if es == 4 else np.uint16) for i in last])
    r = r if es == 4 else mxref.bf16_values(r)
    assert np.array_equal(r, 2 * x[last])
    h, bh = norm_and_bound(r.astype(np.float64), 1, 1e-5, 1.0)
    assert (np.abs(read(8192, k) - h) <= bh + 2 * U * np.abs(h)).all()


def test_offsets_past_32_bits_in_planes(T):
    """planes of more than 4 GiB of codes: written from one row of stride 0, read back, as either operand of a product"""
    rng = np.random.default_rng(5)
    k, rows, m = 8192, (1 << 20) + 5, 16
    x = rng.integers(-6, 7, (1, k)).astype(np.float32)
    x[0, ::32] = 6.0                                           # (every block's scale is 1)
    codes, byte = mxref.quantize(x)
    q = T.mxfp4_quantize(T.to_device(x).view(0, (rows, k), (0, 1)))
    assert q.buf.nbytes > 1 << 32
    one = mxref.planes(codes, byte)
    for i in (0, 1, rows // 2, rows - 2, rows - 1):
        assert np.array_equal(fetch(T, q.buf, i * k // 2, (k // 2,), np.uint8), one[:k // 2])
        assert np.array_equal(fetch(T, q.buf, rows * k // 2 + i * k // 32, (k // 32,), np.uint8), one[k // 2:])
    v = mxref.values(codes, byte)
    wc, wb, _, _ = operands(rng, 1, k, m, True)
    got = T.mul_mat(split(T, wc, wb), q).numpy()
    assert np.array_equal(got, np.repeat((v @ mxref.values(wc, wb).T).astype(np.float32), rows, 0))
    del got
    for n in (3, 40):                                          # rows, then tiles
        b = rng.integers(-8, 9, (n, k)).astype(np.float32)
        got = T.mul_mat(q, dev(T, b, "bf16"), out=T.empty((n, rows + 3)).view(0, (n, rows), (rows + 3, 1)))
        want = (b.astype(np.float64) @ v.T).astype(np.float32)
        for i in (0, n - 1):
            row = fetch(T, got, i * (rows + 3) * 4, (rows,), np.float32)
            assert (row == want[i, 0]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantizer_in_a_graph(T, dtype):
    """quantize, repack and dequantize on a stream of their own, replayed between eager work"""
    rng = np.random.default_rng(6)
    xs = [rng.standard_normal((37, 160)).astype(np.float32) for _ in range(3)]
    if dtype == "bf16":
        xs = [mxref.bf16_values(mxref.bf16_bits(x)) for x in xs]
    st = T.Stream()
    x, q, blk, y = dev(T, xs[0], dtype), T.mxfp4_quantize(dev(T, xs[0], dtype)), T.empty((37, 5, 17), "u8"), T.empty((37, 160))
    T.synchronize()

    def run():
        T.mxfp4_quantize(x, out=q, stream=st)
        T.mxfp4_quantize(x, out=blk, stream=st)
        T.mxfp4_dequantize(q, out=y, stream=st)

    g = T.Graph(st, run)
    for i in (1, 2, 0, 1):
        src = dev(T, xs[i], dtype)
        T._hipcheck(T.hip().hipMemcpy(ctypes.c_void_p(x.ptr), ctypes.c_void_p(src.ptr), x.nbytes, 3), "hipMemcpy D2D")
        T.mxfp4_quantize(dev(T, xs[0], dtype))
        T.synchronize()
        g.launch()
        st.synchronize()
        codes, byte = mxref.quantize(xs[i])
        assert np.array_equal(q.buf.numpy(), mxref.planes(codes, byte))
        assert np.array_equal(blk.numpy(), mxref.blocks(codes, byte))
        assert np.array_equal(y.numpy(), mxref.values(codes, byte).astype(np.float32))
    g.destroy()
    st.destroy()


def test_two_streams_at_once(T):
    """f32 activations rounded and blocks repacked in each stream's own scratch"""
    rng = np.random.default_rng(7)
    n, k, m = 300, 1024, 1024
    streams, work = [T.Stream(), T.Stream()], []
    for s in streams:
        codes, byte = mxref.quantize(rng.standard_normal((m, k)).astype(np.float32))
        w, x = T.to_device(mxref.blocks(codes, byte)), T.to_device(rng.standard_normal((n, k)).astype(np.float32))
        work.append((w, x, T.mul_mat(w, x, a_type=T.MXFP4).numpy(), T.empty((n, m)), s))
    T.synchronize()
    for _ in range(10):
        for w, x, _, out, s in work:
            T.mul_mat(w, x, out=out, a_type=T.MXFP4, stream=s)
    for s in streams:
        s.synchronize()
    for _, _, want, out, _ in work:
        assert np.array_equal(out.numpy(), want)
    for s in streams:
        s.destroy()


def test_bound_workspace(T):
    """exactly what tsk_workspace_size names is enough; less is refused before any launch"""
    rng = np.random.default_rng(8)
    n, k, m = 300, 1024, 1024
    codes, byte = mxref.quantize(rng.standard_normal((m, k)).astype(np.float32))
    w, x = T.to_device(mxref.blocks(codes, byte)), T.to_device(rng.standard_normal((n, k)).astype(np.float32))
    want = T.mul_mat(w, x, a_type=T.MXFP4).numpy()
    st = T.Stream()
    out = T.to_device(np.full((n, m), 5.0, np.float32))
    need = m * k // 32 * 17 + n * k * 2                        # the planes and the rounded rows, 256 bytes apart already
    assert T.workspace_size(T.OP_MUL_MAT, [(w, T.MXFP4), x], out) == need
    small, buf = T.empty((need - 256,), "u8"), T.empty((need,), "u8")
    T.set_workspace(small, stream=st)
    with pytest.raises(T.TskError) as ei:
        T.mul_mat(w, x, out=out, a_type=T.MXFP4, stream=st)
    assert ei.value.status == -9
    st.synchronize()
    assert (out.numpy() == 5.0).all()
    T.set_workspace(buf, stream=st)
    T.mul_mat(w, x, out=out, a_type=T.MXFP4, stream=st)
    st.synchronize()
    assert np.array_equal(out.numpy(), want)
    T.set_workspace(None, stream=st)
    st.destroy()
