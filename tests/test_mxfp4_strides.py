"""Strides of the MXFP4 entry points, checked on the host (no GPU needed): which rows count as evenly spaced where an
extent is broadcast (a stride of 0), and which block tensors are refused for it."""
import ctypes

import pytest

from test_abi import fake, tsk, uninit  # noqa: F401  (fixtures)
from test_mxfp4_abi import ARG, NOT_INIT, STRIDE, call, mx


def strided(T, shape, nb, typ=None, data=0x100000):
    """F32 / BF16 rows of ne = reversed(shape) with the byte strides nb of the outer extents"""
    d = fake(T, T.F32 if typ is None else typ, shape, 2 if typ == T.BF16 else 4)
    d.nb[1], d.nb[2], d.nb[3] = nb
    d.data = data
    return d


def blocks(T, ne, nb, data=0x40000000):
    d = mx(T, 1, ne[0], split=False, data=data)
    for i in range(1, 4):
        d.ne[i], d.nb[i] = ne[i], nb[i - 1]
    return d


def workspace(T, *srcs, dst):
    P = ctypes.POINTER(T.TskTensor)
    arr, n = (P * len(srcs))(*[ctypes.pointer(s) for s in srcs]), ctypes.c_size_t()
    assert T.load().tsk_workspace_size(T.OP_MUL_MAT, arr, len(srcs), ctypes.byref(dst), ctypes.byref(n)) == 0
    return n.value


K, M = 1024, 4096
ROW = 4 * K
# outer extents (ne1, ne2, ne3), byte strides, rows of one product: all of them where they are evenly spaced, else ne1
SPACED = [((100, 3, 1), (ROW, 100 * ROW, 0), 300), ((100, 3, 2), (ROW, 100 * ROW, 300 * ROW), 600),
          ((100, 1, 3), (ROW, 16, 100 * ROW), 300), ((100, 3, 1), (ROW, 200 * ROW, 0), 100),
          # broadcast along the first, the second, the third extent, and along two of them
          ((100, 3, 1), (0, ROW, 0), 100), ((100, 3, 1), (0, ROW, 16), 100), ((100, 3, 2), (0, ROW, 3 * ROW), 100),
          ((100, 3, 1), (ROW, 0, 0), 100), ((100, 3, 2), (ROW, 0, 100 * ROW), 100), ((100, 1, 3), (ROW, 16, 0), 100),
          ((100, 3, 2), (ROW, 100 * ROW, 0), 100), ((100, 1, 3), (0, 16, ROW), 100), ((100, 3, 2), (0, 0, ROW), 100),
          ((100, 3, 2), (0, ROW, 0), 100), ((100, 3, 2), (ROW, 0, 0), 100), ((100, 3, 2), (0, 0, 0), 100)]


@pytest.mark.parametrize("ne,nb,rows", SPACED)
def test_rows_of_one_product(uninit, ne, nb, rows):  # noqa: F811
    """f32 rows of N K M > 2^28 are rounded into scratch, one product's rows at a time: 2 K bytes a row"""
    T = uninit
    x, y = strided(T, ne[::-1] + (K,), nb), fake(T, T.F32, ne[::-1] + (M,), 4)
    assert workspace(T, mx(T, M, K), x, dst=y) == rows * K * 2
    # ... with as few where it is the output whose slices lie apart
    y.nb[2] = y.nb[2] if ne[1] == 1 else y.nb[2] + 64
    y.nb[3] = y.nb[1] * ne[0] + 64 if ne[1] == 1 else y.nb[2] * ne[1]
    if ne[1] * ne[2] > 1:
        assert workspace(T, mx(T, M, K), x, dst=y) == ne[0] * K * 2


# MXFP4 blocks of rows of 64 values (34 bytes): broadcast in one or two extents
BROADCAST = [((64, 7, 2, 1), (0, 34, 0)), ((64, 7, 2, 1), (17, 0, 34)), ((64, 7, 2, 1), (34, 0, 0)), ((64, 7, 2, 3), (0, 34, 68)),
             ((64, 7, 2, 3), (34, 0, 238)), ((64, 7, 2, 3), (34, 238, 0)), ((64, 7, 1, 3), (0, 5, 34)), ((64, 7, 1, 3), (34, 5, 0)),
             ((64, 1, 2, 3), (5, 0, 34)), ((64, 7, 2, 3), (0, 0, 34)), ((64, 7, 2, 3), (0, 0, 0))]


@pytest.mark.parametrize("ne,nb", BROADCAST)
def test_broadcast_blocks(uninit, ne, nb):  # noqa: F811
    """the kernels take blocks in evenly spaced rows: others are refused, as output and as input"""
    T = uninit
    rows = fake(T, T.F32, ne[::-1], 4)
    assert call(T, "tsk_mxfp4_quantize", rows, blocks(T, ne, nb)) == STRIDE
    assert call(T, "tsk_mxfp4_dequantize", blocks(T, ne, nb), rows) == STRIDE


@pytest.mark.parametrize("ne,nb", [((64, 7, 2, 3), (34, 238, 476)), ((64, 7, 2, 3), (40, 280, 560)), ((64, 1, 2, 3), (0, 34, 68)),
                                   ((64, 7, 1, 3), (34, 0, 238)), ((64, 7, 2, 1), (34, 238, 0)), ((64, 1, 1, 1), (0, 0, 0))])
def test_evenly_spaced_blocks(uninit, ne, nb):  # noqa: F811
    """strides of 0 of extents of 1 say nothing"""
    T = uninit
    rows = fake(T, T.F32, ne[::-1], 4)
    assert call(T, "tsk_mxfp4_quantize", rows, blocks(T, ne, nb)) == NOT_INIT
    assert call(T, "tsk_mxfp4_dequantize", blocks(T, ne, nb), rows) == NOT_INIT


def test_columns_beside_broadcast_rows(uninit):  # noqa: F811
    """columns of one array are apart where the rows of an input are broadcast along any extent, and meet where they do"""
    T = uninit
    ld, base = 1024, 0x200000
    y = strided(T, (2, 3, 5, 64), (ld, 5 * ld, 15 * ld), data=base)
    p = T.BlockNormParams(0, 1e-5, None, None, 1.0, T.NORM_LAYER, 1e-5, None, None, None)
    for nb in ((0, 5 * ld, 15 * ld), (ld, 0, 15 * ld), (ld, 5 * ld, 0), (0, 0, 15 * ld), (ld, 0, 0), (0, 5 * ld, 0)):
        for at in (256, 768, -256):
            assert call(T, "tsk_block_norm", strided(T, (2, 3, 5, 64), nb, data=base + at), None, p, None, y) == NOT_INIT
        for at in (252, 0, -252, 772):
            assert call(T, "tsk_block_norm", strided(T, (2, 3, 5, 64), nb, data=base + at), None, p, None, y) == ARG
