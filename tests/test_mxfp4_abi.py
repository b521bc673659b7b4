"""Refusals of the MXFP4 entry points and of the block norm: every bad operand
is turned down on the host, before any launch, with the status that names it
(no GPU needed)."""
import ctypes

import numpy as np
import pytest

import mxref
from test_abi import fake, tsk, uninit  # noqa: F401  (fixtures)

NOT_INIT, ARG, TYPE, SHAPE, STRIDE, ALIGN, UNSUP = -7, -1, -2, -3, -4, -5, -6


def mx(T, rows, k, split=True, data=0x40000000):
    d = T.TskTensor()
    d.type = T.MXFP4_SPLIT if split else T.MXFP4
    d.ne[0], d.ne[1], d.ne[2], d.ne[3] = k, rows, 1, 1
    d.nb[0], d.nb[1] = (1, k) if split else (17, k // 32 * 17)
    d.nb[2] = d.nb[3] = d.nb[1] * rows
    d.data = data
    return d


def call(T, fn, *args):
    return getattr(T.load(), fn)(*[ctypes.byref(a) if isinstance(a, ctypes.Structure) else a for a in args], None)


def test_split_nbytes(tsk):  # noqa: F811
    lib = tsk.load()
    assert lib.tsk_mxfp4_split_nbytes(64, 3) == 3 * 32 + 3 * 2
    assert lib.tsk_mxfp4_split_nbytes(40, 3) == 0 and lib.tsk_mxfp4_split_nbytes(32, 0) == 0
    assert lib.tsk_mxfp4_split_nbytes(1 << 17, 1 << 17) == (1 << 34) // 32 * 17


def test_quantize_refusals(uninit):  # noqa: F811
    T = uninit
    x = fake(T, T.F32, (77, 1024), 4)
    assert call(T, "tsk_mxfp4_quantize", x, mx(T, 77, 1024)) == NOT_INIT
    assert call(T, "tsk_mxfp4_quantize", x, mx(T, 77, 1024, split=False)) == NOT_INIT
    assert call(T, "tsk_mxfp4_quantize", fake(T, T.BF16, (77, 1024), 2), mx(T, 77, 1024)) == NOT_INIT
    assert call(T, "tsk_mxfp4_quantize", x, None) == ARG
    assert call(T, "tsk_mxfp4_quantize", fake(T, T.F16, (77, 1024), 2), mx(T, 77, 1024)) == TYPE
    assert call(T, "tsk_mxfp4_quantize", x, fake(T, T.Q8_0, (77, 1024), 34)) == TYPE
    assert call(T, "tsk_mxfp4_quantize", x, mx(T, 76, 1024)) == SHAPE
    assert call(T, "tsk_mxfp4_quantize", fake(T, T.F32, (77, 1000), 4), mx(T, 77, 1000)) == SHAPE
    odd = fake(T, T.F32, (77, 1024), 4)
    odd.nb[0] = 8
    assert call(T, "tsk_mxfp4_quantize", odd, mx(T, 77, 1024)) == STRIDE
    bad = mx(T, 77, 1024, split=False)
    bad.nb[0] = 18
    assert call(T, "tsk_mxfp4_quantize", x, bad) == STRIDE
    bad = mx(T, 77, 1024, split=False)
    bad.nb[1] -= 1                                             # rows that overlap
    assert call(T, "tsk_mxfp4_quantize", x, bad) == STRIDE
    assert call(T, "tsk_mxfp4_quantize", x, mx(T, 77, 1024, data=0x40000008)) == ALIGN
    assert call(T, "tsk_mxfp4_quantize", x, mx(T, 77, 1024, data=x.data)) == ARG     # in place
    x.data += 2
    assert call(T, "tsk_mxfp4_quantize", x, mx(T, 77, 1024)) == ALIGN


def test_dequantize_and_repack_refusals(uninit):  # noqa: F811
    T = uninit
    y = fake(T, T.F32, (5, 64), 4)
    assert call(T, "tsk_mxfp4_dequantize", mx(T, 5, 64), y) == NOT_INIT
    assert call(T, "tsk_mxfp4_dequantize", mx(T, 5, 64, split=False), fake(T, T.BF16, (5, 64), 2)) == NOT_INIT
    assert call(T, "tsk_mxfp4_dequantize", fake(T, T.F32, (5, 64), 4), y) == TYPE
    assert call(T, "tsk_mxfp4_dequantize", mx(T, 5, 64), fake(T, T.I32, (5, 64), 4)) == TYPE
    assert call(T, "tsk_mxfp4_dequantize", mx(T, 5, 96), y) == SHAPE
    assert call(T, "tsk_mxfp4_dequantize", mx(T, 5, 64, data=y.data + 16), y) == ARG
    assert call(T, "tsk_mxfp4_repack", mx(T, 5, 64, split=False), mx(T, 5, 64, data=0x50000000)) == NOT_INIT
    assert call(T, "tsk_mxfp4_repack", mx(T, 5, 64), mx(T, 5, 64)) == TYPE
    assert call(T, "tsk_mxfp4_repack", mx(T, 5, 64, split=False), mx(T, 4, 64, data=0x50000000)) == SHAPE
    assert call(T, "tsk_mxfp4_repack", mx(T, 5, 64, split=False), mx(T, 5, 64)) == ARG     # the same bytes


def test_mul_mat_refusals(uninit):  # noqa: F811
    T = uninit
    mm = lambda a, b, d, bias=None: call(T, "tsk_mul_mat", a, b, bias, d)
    w, x, y = mx(T, 96, 64), fake(T, T.F32, (7, 64), 4), fake(T, T.F32, (7, 96), 4)
    for b in (x, fake(T, T.BF16, (7, 64), 2), mx(T, 7, 64)):
        assert mm(w, b, y) == NOT_INIT and mm(mx(T, 96, 64, split=False), b, y) == NOT_INIT
        assert call(T, "tsk_mul_mat_noalloc", w, b, None, y) == NOT_INIT
    assert mm(w, fake(T, T.F16, (7, 64), 2), y) == TYPE
    assert mm(w, mx(T, 7, 64, split=False), y) == TYPE          # activations come as planes
    assert mm(fake(T, T.BF16, (96, 64), 2), mx(T, 7, 64), y) == TYPE
    assert mm(w, x, fake(T, T.F16, (7, 96), 2)) == TYPE
    assert mm(mx(T, 96, 48), fake(T, T.F32, (7, 48), 4), y) == SHAPE
    assert mm(w, mx(T, 7, 96), y) == SHAPE
    assert mm(w, mx(T, 8, 64), y) == SHAPE
    assert mm(w, mx(T, 7, 64, data=0x40000004), y) == ALIGN
    assert mm(mx(T, 96, 64, data=0x40000004), x, y) == ALIGN
    odd = fake(T, T.F32, (7, 97), 4)                            # rows of 388 bytes
    assert mm(mx(T, 97, 64), x, odd) == ALIGN
    odd.nb[1] = 400
    odd.nb[2] = odd.nb[3] = 2800
    assert mm(mx(T, 97, 64), x, odd) == NOT_INIT
    assert mm(w, x, y, fake(T, T.F32, (95,), 4)) == SHAPE


def test_mul_mat_workspace(uninit):  # noqa: F811
    T = uninit

    def ws(*srcs, dst):
        P = ctypes.POINTER(T.TskTensor)
        arr, n = (P * len(srcs))(*[ctypes.pointer(s) for s in srcs]), ctypes.c_size_t()
        rc = T.load().tsk_workspace_size(T.OP_MUL_MAT, arr, len(srcs), ctypes.byref(dst), ctypes.byref(n))
        ok = T.load().tsk_supports_op(T.OP_MUL_MAT, arr, len(srcs), ctypes.byref(dst))
        assert (rc == 0) == (ok == 1)
        return rc, n.value

    x, y = fake(T, T.F32, (7, 64), 4), fake(T, T.F32, (7, 96), 4)
    # blocks are repacked into scratch: their planes, rounded up to 256 bytes
    assert ws(mx(T, 96, 64, split=False), x, dst=y) == (0, (96 * 34 + 255) // 256 * 256)
    assert ws(mx(T, 96, 64), mx(T, 7, 96), dst=y)[0] == SHAPE


def params(T, **kw):
    p = T.BlockNormParams(0, 1e-5, None, None, 1.0, T.NORM_LAYER, 1e-5, None, None, None)
    keep = []
    for k, v in kw.items():
        if isinstance(v, T.TskTensor):
            keep.append(v)
            v = ctypes.pointer(v)
        setattr(p, k, v)
    p._keep = keep
    return p


def test_block_norm_refusals(uninit):  # noqa: F811
    T = uninit
    t = lambda shape, typ=None, data=0x100000: _at(fake(T, T.F32 if typ is None else typ, shape,
                                                        2 if typ == T.BF16 else 4), data)

    def _at(d, data):
        d.data = data
        return d

    S = (2, 7, 64)
    x, y = t(S), t(S, data=0x200000)
    res, dst = t(S, data=0x300000), t(S, data=0x400000)
    bn = lambda x, y, p, res, dst: call(T, "tsk_block_norm", x, y, p, res, dst)
    f = lambda shape, data=0x500000: t(shape, data=data)
    assert bn(x, y, params(T), res, dst) == NOT_INIT
    assert bn(x, None, params(T), None, dst) == NOT_INIT
    assert bn(x, y, params(T, pre_norm=0), res, None) == NOT_INIT
    assert bn(x, y, params(T), x, dst) == NOT_INIT              # in place
    for shape in ((64,), (1, 1, 64), (2, 1, 64), (2, 7, 64)):
        assert bn(x, y, params(T, gate=f(shape), scale=f(shape, 0x600000), shift=f(shape, 0x700000)), res, dst) == NOT_INIT
    m = mx(T, 14, 64)
    m.ne[1], m.ne[2] = 7, 2
    assert bn(x, y, params(T), res, m) == NOT_INIT
    assert bn(x, y, None, res, dst) == ARG
    assert bn(x, y, params(T), None, None) == ARG
    assert bn(x, y, params(T), res, None) == ARG                # a norm without its output
    assert bn(x, None, params(T, gate=f((64,))), res, dst) == ARG
    assert bn(x, None, params(T, post_norm=1), res, dst) == ARG
    assert bn(x, None, params(T, post_w=f((64,))), res, dst) == ARG
    assert bn(x, y, params(T, pre_norm=3), res, dst) == ARG
    assert bn(x, y, params(T, pre_eps=float("nan")), res, dst) == ARG
    assert bn(x, y, params(T, post_eps=-1.0), res, dst) == ARG
    assert bn(x, y, params(T, res_scale=float("nan")), res, dst) == ARG
    assert bn(t(S, T.F16), y, params(T), res, dst) == TYPE
    assert bn(x, y, params(T), t(S, T.BF16, 0x300000), dst) == TYPE     # res in another type than x
    assert bn(x, y, params(T), res, t(S, T.BF16, 0x400000)) == NOT_INIT
    assert bn(x, t((2, 6, 64), data=0x200000), params(T), res, dst) == SHAPE
    assert bn(x, y, params(T, gate=f((2, 3, 64))), res, dst) == SHAPE
    assert bn(x, y, params(T, gate=f((1,))), res, dst) == SHAPE
    assert bn(x, y, params(T, scale=t((64,), T.BF16)), res, dst) == TYPE
    assert bn(x, y, params(T, pre_w=f((63,))), res, dst) == SHAPE
    assert bn(x, y, params(T), res, mx(T, 14, 64)) == SHAPE
    assert bn(t((2, 7, 40)), None, params(T), None, mx(T, 14, 40)) == SHAPE
    strided = t(S)
    strided.nb[0] = 8
    assert bn(strided, y, params(T), res, dst) == STRIDE
    assert bn(x, y, params(T), t(S, data=0x300002), dst) == ALIGN
    # outputs over inputs or each other
    assert bn(x, y, params(T), res, x) == ARG
    assert bn(x, y, params(T), y, dst) == ARG
    assert bn(x, y, params(T), res, res) == ARG
    assert bn(x, y, params(T), t(S, data=x.data + 4), dst) == ARG
    assert bn(x, y, params(T, gate=f((64,), dst.data + 256)), res, dst) == ARG
    # columns of one array side by side are apart
    wide = []
    for i in range(2):
        d = t(S, data=0x800000 + 256 * i)
        d.nb[1], d.nb[2], d.nb[3] = 512, 512 * 7, 512 * 14
        wide.append(d)
    assert bn(wide[0], y, params(T), wide[1], dst) == NOT_INIT
    wide[1].data -= 4
    assert bn(wide[0], y, params(T), wide[1], dst) == ARG


def test_outputs_whose_rows_share_bytes(uninit):  # noqa: F811
    """rows of an output that overlap, strides of extents of 1 aside; broadcast inputs are taken"""
    T = uninit

    def strided(shape, nb, typ=None, data=0x100000):
        d = fake(T, T.F32 if typ is None else typ, shape, 2 if typ == T.BF16 else 4)
        d.nb[1], d.nb[2], d.nb[3] = nb
        d.data = data
        return d

    S, B = (2, 7, 64), 256                                      # rows of 256 bytes
    q = mx(T, 14, 64, data=0x800000)
    q.ne[1], q.ne[2] = 7, 2
    good, bad = [(B, 7 * B, 0), (2 * B, B, 0), (B + 4, 8 * B, 1)], [(0, 7 * B, 0), (B, 0, 0), (B, 6 * B, 0), (B - 4, 7 * B, 0)]
    for nb in good:                                             # the second: two interleaved sets of rows
        assert call(T, "tsk_mxfp4_dequantize", q, strided(S, nb)) == NOT_INIT
    w, x = mx(T, 64, 64), strided(S, (0, 0, 0), data=0x300000)
    for nb in bad:
        assert call(T, "tsk_mxfp4_dequantize", q, strided(S, nb)) == STRIDE
        y, other = strided(S, nb, data=0x100000), strided(S, (B, 7 * B, 0), data=0x200000)
        p = params(T)
        for res, dst in ((y, other), (other, y)):
            assert call(T, "tsk_block_norm", x, None, p, res, dst) == STRIDE
        if nb[0] % 16 == 0:
            assert call(T, "tsk_mul_mat", w, x, None, y) == STRIDE
    in_place = strided(S, (0, 7 * B, 0))
    assert call(T, "tsk_block_norm", in_place, None, params(T, pre_norm=0), in_place, None) == STRIDE
    assert call(T, "tsk_block_norm", x, None, params(T), None, strided(S, (B, 7 * B, 0))) == NOT_INIT
    assert call(T, "tsk_mul_mat", w, x, None, strided(S, (B, 7 * B, 0))) == NOT_INIT
    # blocks: rows along the third extent alone
    x = strided((3, 1, 1, 64), (4, 4, B), data=0x300000)
    for nb, rc in (((3, 5, 34), NOT_INIT), ((34, 34, 33), STRIDE), ((34, 34, 0), STRIDE)):
        d = mx(T, 1, 64, split=False, data=0x800000)
        d.ne[3] = 3
        d.nb[1], d.nb[2], d.nb[3] = nb
        assert call(T, "tsk_mxfp4_quantize", x, d) == rc
        assert call(T, "tsk_mxfp4_dequantize", d, strided((3, 1, 1, 64), (4, 4, B))) == rc


def test_planes_of_too_few_bytes(tsk):  # noqa: F811
    tsk.SplitMXFP4(np.zeros(4 * 34, np.uint8), 64, 4)
    with pytest.raises(ValueError):
        tsk.SplitMXFP4(np.zeros(4 * 34 - 1, np.uint8), 64, 4)


def test_reference_rounding():
    """the 64-bit restatement itself: the numbers, the ties and the ends of the scale"""
    top = 7.9
    x = np.zeros((1, 32), np.float32)
    x[0, :16] = [top, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, 0.26, 5.01, -7.0, 0.0, -0.0, 6.0, 0.24]
    c, b = mxref.quantize(x)
    assert b[0, 0] == 127
    assert c[0, :16].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 8, 1, 7, 15, 0, 8, 7, 0]
    x = np.zeros((5, 32), np.float32)
    x[1, 3] = 2.0 ** -149
    x[2, 3] = np.inf
    x[3, 0] = np.nan
    x[4, 0] = np.finfo(np.float32).max
    c, b = mxref.quantize(x)
    assert b[:, 0].tolist() == [0, 0, 255, 255, 252] and c[4, 0] == 7
    v = mxref.values(c, b)
    assert np.isnan(v[2:4]).all() and v[4, 0] == 6 * 2.0 ** 125
    c2, b2 = mxref.unplanes(mxref.planes(c, b), 5, 32)
    assert (c2 == c).all() and (b2 == b).all()
    assert mxref.blocks(c, b).shape == (5, 1, 17)


@pytest.mark.parametrize("v", [1.0, 1.5, 3.9999998, 4.0, 2.0 ** -126])
def test_reference_scale(v):
    x = np.full((1, 32), v, np.float32)
    c, b = mxref.quantize(x)
    assert int(b[0, 0]) - 127 == max(int(np.floor(np.log2(np.float64(np.float32(v))))) - 2, -127)
