"""Refusals of the 8-bit rows, of the rotary positions over several axes and of
cross attention: every bad operand is turned down on the host, before any
launch, with the status that names it (no GPU needed)."""
import ctypes

import numpy as np
import pytest

import crossref
from test_abi import fake, tsk, uninit  # noqa: F401  (fixtures)
from test_mxfp4_abi import call, params as bn_params

NOT_INIT, ARG, TYPE, SHAPE, STRIDE, ALIGN, UNSUP = -7, -1, -2, -3, -4, -5, -6


def i8(T, rows, k, data=0x40000000):
    d = T.TskTensor()
    d.type = T.I8_SPLIT
    d.ne[0], d.ne[1], d.ne[2], d.ne[3] = k, rows, 1, 1
    d.nb[0], d.nb[1], d.nb[2], d.nb[3] = 1, k, 0, 0
    d.data = data
    return d


def at(d, data):
    d.data = data
    return d


def test_split_nbytes(tsk):  # noqa: F811
    lib = tsk.load()
    assert lib.tsk_i8_split_nbytes(64, 3) == 3 * 64 + 12
    assert lib.tsk_i8_split_nbytes(65, 3) == 3 * 80 + 12
    assert lib.tsk_i8_split_nbytes(0, 3) == 0 and lib.tsk_i8_split_nbytes(32, 0) == 0
    assert lib.tsk_i8_split_nbytes(1 << 17, 1 << 17) == (1 << 34) + (1 << 19)
    with pytest.raises(ValueError):
        tsk.SplitI8(np.zeros(3 * 80 + 11, np.uint8), 65, 3)
    tsk.SplitI8(np.zeros(3 * 80 + 12, np.uint8), 65, 3)


def test_quantize_refusals(uninit):  # noqa: F811
    T = uninit
    x = fake(T, T.F32, (77, 1000), 4)
    quant = lambda x, y: call(T, "tsk_i8_quantize", x, y)
    deq = lambda x, y: call(T, "tsk_i8_dequantize", x, y)
    for t, es in ((T.F32, 4), (T.BF16, 2)):
        assert quant(fake(T, t, (77, 1000), es), i8(T, 77, 1000)) == NOT_INIT
        assert deq(i8(T, 77, 1000), fake(T, t, (77, 1000), es)) == NOT_INIT
        assert quant(fake(T, t, (1, 1), es), i8(T, 1, 1)) == NOT_INIT
    assert quant(x, None) == ARG
    assert quant(fake(T, T.F16, (77, 1000), 2), i8(T, 77, 1000)) == TYPE
    assert deq(i8(T, 77, 1000), fake(T, T.F16, (77, 1000), 2)) == TYPE
    assert quant(x, fake(T, T.F32, (77, 1000), 4)) == TYPE
    assert deq(fake(T, T.F32, (77, 1000), 4), x) == TYPE
    assert quant(x, i8(T, 76, 1000)) == SHAPE and deq(i8(T, 77, 1001), x) == SHAPE
    big = i8(T, 1, 1000)
    big.ne[1], big.ne[2] = 1 << 20, 1 << 20
    assert deq(big, x) == SHAPE
    odd = fake(T, T.F32, (77, 1000), 4)
    odd.nb[0] = 8
    assert quant(odd, i8(T, 77, 1000)) == STRIDE and deq(i8(T, 77, 1000), odd) == STRIDE
    assert quant(x, i8(T, 77, 1000, 0x40000008)) == ALIGN
    assert quant(x, i8(T, 77, 1000, x.data)) == ARG
    # the scales end past the integers: 77 * (1008 + 4) bytes
    assert deq(i8(T, 77, 1000, 0x40000000), at(fake(T, T.F32, (77, 1000), 4), 0x40000000 + 77 * 1012 - 4)) == ARG
    assert deq(i8(T, 77, 1000, 0x40000000), at(fake(T, T.F32, (77, 1000), 4), 0x40000000 + 77 * 1012)) == NOT_INIT
    overlapping = fake(T, T.F32, (77, 1000), 4)
    overlapping.nb[1] = 3996
    assert deq(i8(T, 77, 1000), overlapping) == STRIDE
    assert quant(overlapping, i8(T, 77, 1000)) == NOT_INIT      # inputs may


def test_mul_mat_refusals(uninit):  # noqa: F811
    T = uninit
    mm = lambda a, b, d, bias=None: call(T, "tsk_mul_mat", a, b, bias, d)
    w, x, y = i8(T, 96, 72), fake(T, T.F32, (7, 72), 4), at(fake(T, T.F32, (7, 96), 4), 0x200000)
    for b in (x, fake(T, T.BF16, (7, 72), 2), i8(T, 7, 72)):
        assert mm(w, b, y) == NOT_INIT
        assert call(T, "tsk_mul_mat_noalloc", w, b, None, y) == NOT_INIT
        assert mm(w, b, at(fake(T, T.BF16, (7, 96), 2), 0x200000)) == NOT_INIT
    for k in (1, 5, 16, 131071):
        assert mm(i8(T, 96, k), i8(T, 7, k), y) == NOT_INIT
    assert mm(i8(T, 96, 131072), i8(T, 7, 131072), y) == SHAPE
    assert mm(w, fake(T, T.F16, (7, 72), 2), y) == TYPE
    assert mm(fake(T, T.BF16, (96, 72), 2), i8(T, 7, 72), y) == TYPE
    assert mm(w, x, at(fake(T, T.F16, (7, 96), 2), 0x200000)) == TYPE
    assert mm(w, i8(T, 7, 73), y) == SHAPE and mm(w, i8(T, 8, 72), y) == SHAPE
    assert mm(w, i8(T, 7, 72, 0x40000004), y) == ALIGN and mm(i8(T, 96, 72, 0x40000004), x, y) == ALIGN
    assert mm(i8(T, 97, 72), x, at(fake(T, T.F32, (7, 97), 4), 0x200000)) == ALIGN     # rows of 388 bytes
    assert mm(w, x, y, fake(T, T.F32, (95,), 4)) == SHAPE
    y.nb[1] = 368
    assert mm(w, x, y) == STRIDE


def test_mul_mat_workspace(uninit):  # noqa: F811
    T = uninit
    P = ctypes.POINTER(T.TskTensor)

    def ws(op, *srcs, dst):
        arr, n = (P * len(srcs))(*[ctypes.pointer(s) for s in srcs]), ctypes.c_size_t()
        rc = T.load().tsk_workspace_size(op, arr, len(srcs), ctypes.byref(dst), ctypes.byref(n))
        ok = T.load().tsk_supports_op(op, arr, len(srcs), ctypes.byref(dst))
        assert (rc == 0) == (ok == 1)
        return rc, n.value

    y = fake(T, T.F32, (7, 96), 4)
    assert ws(T.OP_MUL_MAT, i8(T, 96, 72), fake(T, T.F32, (7, 72), 4), dst=y) == (0, (7 * 84 + 255) // 256 * 256)
    assert ws(T.OP_MUL_MAT, i8(T, 96, 72), i8(T, 7, 72), dst=y) == (0, 0)
    assert ws(T.OP_MUL_MAT, i8(T, 96, 72), i8(T, 7, 71), dst=y)[0] == SHAPE
    q, k = fake(T, T.BF16, (2, 8, 5, 64), 2), fake(T, T.BF16, (2, 2, 300, 64), 2)
    assert ws(T.OP_CROSS_ATTENTION, q, k, k, dst=fake(T, T.BF16, (2, 5, 8, 64), 2))[0] == 0
    assert ws(T.OP_CROSS_ATTENTION, q, k, k, dst=fake(T, T.BF16, (2, 8, 5, 64), 2))[0] == SHAPE


def test_block_norm_takes_8_bit_rows(uninit):  # noqa: F811
    T = uninit
    x = at(fake(T, T.F32, (2, 7, 40), 4), 0x100000)
    res = at(fake(T, T.F32, (2, 7, 40), 4), 0x300000)
    d = i8(T, 7, 40)
    d.ne[2] = 2
    assert call(T, "tsk_block_norm", x, None, bn_params(T), res, d) == NOT_INIT
    assert call(T, "tsk_block_norm", x, None, bn_params(T), None, at(d, x.data + 64)) == ARG
    assert call(T, "tsk_block_norm", x, None, bn_params(T), None, at(d, 0x40000008)) == ALIGN
    assert call(T, "tsk_block_norm", x, None, bn_params(T), None, i8(T, 14, 40)) == SHAPE


def rope_params(T, dims=(32, 16, 16), **kw):
    p = T.RopeAxesParams(len(dims), (ctypes.c_int * 4)(*dims[:4]), 0, 0, 10000.0, 1.0, None, 1e-6)
    for k, v in kw.items():
        if isinstance(v, T.TskTensor):
            p._keep, v = v, ctypes.pointer(v)
        setattr(p, k, v)
    return p


def test_rope_axes_refusals(uninit):  # noqa: F811
    T = uninit
    x = at(fake(T, T.F32, (2, 7, 3, 64), 4), 0x100000)
    y = at(fake(T, T.BF16, (2, 7, 3, 64), 2), 0x200000)
    pos = at(fake(T, T.I32, (3, 7), 4), 0x300000)
    rope = lambda x, pos, p, y: call(T, "tsk_rope_axes", x, pos, p, y)
    P = lambda *a, **kw: rope_params(T, *a, **kw)
    assert rope(x, pos, P(), y) == NOT_INIT and rope(x, pos, P(), x) == NOT_INIT
    assert rope(x, at(fake(T, T.F32, (2, 3, 7), 4), 0x300000), P(pairs=1, shared_freqs=1), y) == NOT_INIT
    assert rope(x, at(fake(T, T.F32, (1, 7), 4), 0x300000), P((64,)), y) == NOT_INIT
    assert rope(x, pos, P((0, 2, 0)), y) == NOT_INIT
    assert rope(x, pos, P(w=at(fake(T, T.F32, (64,), 4), 0x400000)), y) == NOT_INIT
    assert rope(x, pos, None, y) == ARG and rope(x, None, P(), y) == ARG
    for dims in ((31, 16, 16), (34, 16, 16), (0, 0, 0), (66, 0, 0), (-2, 16, 16)):
        assert rope(x, pos, P(dims), y) == ARG
    assert rope(x, pos, P((8, 8, 8, 8), n_axes=5), y) == ARG and rope(x, pos, P(n_axes=0), y) == ARG
    assert rope(x, pos, P(pairs=2), y) == ARG
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        assert rope(x, pos, P(freq_base=bad), y) == ARG
    assert rope(x, pos, P(freq_scale=float("nan")), y) == ARG
    assert rope(x, pos, P(w=at(fake(T, T.F32, (64,), 4), 0x400000), eps=-1.0), y) == ARG
    assert rope(x, pos, P(w=at(fake(T, T.F32, (63,), 4), 0x400000)), y) == SHAPE
    assert rope(x, pos, P((32, 16)), y) == SHAPE                # positions on another number of axes
    assert rope(x, at(fake(T, T.I32, (3, 6), 4), 0x300000), P(), y) == SHAPE
    assert rope(x, at(fake(T, T.I32, (3, 3, 7), 4), 0x300000), P(), y) == SHAPE
    assert rope(x, at(fake(T, T.BF16, (3, 7), 2), 0x300000), P(), y) == TYPE
    assert rope(at(fake(T, T.F16, (2, 7, 3, 64), 2), 0x100000), pos, P(), y) == TYPE
    assert rope(x, pos, P(), at(fake(T, T.F32, (2, 7, 3, 32), 4), 0x200000)) == SHAPE
    wide = at(fake(T, T.F32, (1, 1, 1, 386), 4), 0x100000)
    assert rope(wide, at(fake(T, T.I32, (3, 1), 4), 0x300000), P(), at(fake(T, T.F32, (1, 1, 1, 386), 4), 0x200000)) == UNSUP
    assert rope(x, pos, P(), at(fake(T, T.BF16, (2, 7, 3, 64), 2), x.data)) == ARG      # another type in the same place
    assert rope(x, pos, P(), at(fake(T, T.F32, (2, 7, 3, 64), 4), x.data + 4)) == ARG
    assert rope(x, at(pos, y.data), P(), y) == ARG
    at(pos, 0x300000)
    s = at(fake(T, T.F32, (2, 7, 3, 64), 4), 0x200000)
    s.nb[1] = 0
    assert rope(x, pos, P(), s) == STRIDE
    pos.nb[0] = 8
    assert rope(x, pos, P(), y) == STRIDE


def cross_params(T, **kw):
    p = T.CrossAttnParams(0.125, None, None, None, 0)
    p._keep = list(kw.values())
    for k, v in kw.items():
        setattr(p, k, ctypes.pointer(v) if isinstance(v, T.TskTensor) else v)
    return p


def test_cross_attention_refusals(uninit):  # noqa: F811
    T = uninit
    B, H, G, N, M, D = 2, 8, 2, 5, 300, 72
    q = at(fake(T, T.BF16, (B, H, N, D), 2), 0x100000)
    k, v = (at(fake(T, T.BF16, (B, G, M, D), 2), a) for a in (0x1000000, 0x2000000))
    y = at(fake(T, T.F32, (B, N, H, D), 4), 0x3000000)
    lens = at(fake(T, T.I32, (B,), 4), 0x4000000)
    P = lambda **kw: cross_params(T, **kw)
    go = lambda q, k, v, p, y: call(T, "tsk_cross_attention", q, k, v, p, y)
    assert go(q, k, v, P(), y) == NOT_INIT
    assert go(q, k, v, P(kv_len=lens, q_len=lens, kv_valid=0x5000000, kv_valid_nb=M), y) == NOT_INIT
    for t, es in ((T.F32, 4), (T.F16, 2)):
        assert go(at(fake(T, t, (B, H, N, D), es), 0x100000), k, v, P(), at(fake(T, t, (B, N, H, D), es), 0x3000000)) == NOT_INIT
    assert go(q, k, v, None, y) == ARG
    assert go(q, k, v, P(scale=0.0), y) == ARG and go(q, k, v, P(scale=float("nan")), y) == ARG
    assert go(q, k, v, P(kv_valid=0x5000000, kv_valid_nb=-1), y) == ARG
    f32 = at(fake(T, T.F32, (B, G, M, D), 4), 0x1000000)
    assert go(q, f32, f32, P(), y) == TYPE
    assert go(q, k, at(fake(T, T.F16, (B, G, M, D), 2), 0x2000000), P(), y) == TYPE
    assert go(q, k, v, P(kv_len=at(fake(T, T.F32, (B,), 4), 0x4000000)), y) == TYPE
    assert go(q, k, v, P(q_len=at(fake(T, T.I32, (B + 1,), 4), 0x4000000)), y) == SHAPE
    assert go(q, k, at(fake(T, T.BF16, (B, G, M - 1, D), 2), 0x2000000), P(), y) == SHAPE
    k3 = at(fake(T, T.BF16, (B, 3, M, D), 2), 0x1000000)
    assert go(q, k3, k3, P(), y) == SHAPE
    k1 = at(fake(T, T.BF16, (1, G, M, D), 2), 0x1000000)
    assert go(q, k1, k1, P(), y) == SHAPE
    assert go(q, k, v, P(), at(fake(T, T.F32, (B, H, N, D), 4), 0x3000000)) == SHAPE
    for d in (136, 60):
        qq, kk = at(fake(T, T.BF16, (1, 1, 1, d), 2), 0x100000), at(fake(T, T.BF16, (1, 1, 8, d), 2), 0x1000000)
        assert go(qq, kk, kk, P(), at(fake(T, T.F32, (1, 1, 1, d), 4), 0x3000000)) == UNSUP
    assert go(at(fake(T, T.BF16, (B, H, N, D), 2), 0x100008), k, v, P(), y) == ALIGN
    for nb in (0, 2 * D - 16, (1 << 24) + 16):
        bad = at(fake(T, T.BF16, (B, G, M, D), 2), 0x1000000)
        bad.nb[1] = nb
        assert go(q, bad, v, P(), y) == STRIDE
    assert go(q, k, v, P(), at(fake(T, T.BF16, (B, N, H, D), 2), q.data)) == ARG
    assert go(q, k, v, P(kv_len=at(lens, y.data)), y) == ARG
    span = B * N * H * D * 4
    assert go(q, k, v, P(kv_valid=y.data - M - 1, kv_valid_nb=M), y) == ARG            # (the second sequence's flags)
    assert go(q, k, v, P(kv_valid=y.data + span - 1), y) == ARG
    assert go(q, k, v, P(kv_valid=y.data - 2 * M, kv_valid_nb=M), y) == NOT_INIT and go(q, k, v, P(kv_valid=y.data + span), y) == NOT_INIT
    rows = at(fake(T, T.F32, (B, N, H, D), 4), 0x3000000)
    rows.nb[2] = 16
    assert go(q, k, v, P(), rows) == STRIDE
    # the states of all sequences in one place, heads broadcast: strides of 0
    k.nb[2] = k.nb[3] = 0
    at(lens, 0x4000000)
    assert go(q, k, v, P(kv_len=lens), y) == NOT_INIT


def test_reference_rounding():
    """the 64-bit restatement itself: ties, zeros, what is not finite"""
    x = np.zeros((5, 20), np.float32)
    x[0, :6] = [127.0, 0.5, 1.5, 2.5, -0.5, -126.5]            # a scale of 1: ties
    x[1, :3] = [381.0, 4.5, 7.5]                               # of 3
    x[2, 3], x[3, 19] = np.inf, np.nan
    q, d = crossref.i8_quantize(x)
    assert q[0, :6].tolist() == [127, 0, 2, 2, 0, -126] and d[0] == 1
    assert q[1, :3].tolist() == [127, 2, 2] and d[1] == 3
    assert np.isnan(d[2:4]).all() and not q[2:].any() and d[4] == np.float32(2.0 ** -100) / np.float32(127)
    p, s = crossref.i8_unplanes(crossref.i8_planes(q, d), 5, 20)
    assert p.shape == (5, 32) and (p[:, :20] == q).all() and not p[:, 20:].any() and np.array_equal(s, d, equal_nan=True)


def test_reference_turn():
    """a quarter turn of every pair, in both arrangements"""
    x = np.arange(1.0, 9).reshape(1, 1, 1, 8)
    out, size = crossref.turn(x, np.full((1, 1, 1), np.pi / 2), [2], False, False)
    assert np.allclose(out[0, 0, 0], [-2, 1, 3, 4, 5, 6, 7, 8]) and size[0, 0, 0, 0] == 3 and size[0, 0, 0, 2] == 0
    out, _ = crossref.turn(x, np.full((1, 2, 1), np.pi / 2), [2, 2], True, False)
    assert np.allclose(out[0, 0, 0], [-3, -4, 1, 2, 5, 6, 7, 8])
