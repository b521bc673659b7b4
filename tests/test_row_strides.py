"""Rows that lie along the outermost extent with gaps between its items, where the extent between has one element (its
stride says nothing): not evenly spaced rows (no GPU needed)."""
import ctypes

import pytest

from test_abi import fake, tsk, uninit  # noqa: F401  (fixtures)

NOT_INIT, STRIDE = -7, -4
ROW = 4 * 1024


def rows(T, ne, nb, data=0x100000):
    """F32 rows of 1024 values, outer extents ne, their byte strides nb"""
    d = fake(T, T.F32, ne[::-1] + (1024,), 4)
    d.nb[1], d.nb[2], d.nb[3] = nb
    d.data = data
    return d


# extents, strides, rows of one product
LAYOUTS = [((6, 1, 3), (ROW, 6 * ROW, 6 * ROW), 18), ((6, 1, 3), (ROW, 16, 6 * ROW), 18), ((6, 2, 3), (ROW, 6 * ROW, 12 * ROW), 36),
           ((6, 1, 3), (ROW, 12 * ROW, 12 * ROW), 6), ((6, 1, 3), (ROW, 6 * ROW, 12 * ROW), 6), ((6, 1, 3), (ROW, ROW, ROW), 6),
           ((1, 1, 3), (ROW, ROW, ROW), 3), ((1, 1, 3), (ROW, 2 * ROW, 2 * ROW), 1), ((1, 3, 1), (ROW, 2 * ROW, 6 * ROW), 1),
           ((6, 1, 3), (ROW, 0, 0), 6)]


@pytest.mark.parametrize("ne,nb,n", LAYOUTS)
def test_rows_of_one_product(uninit, ne, nb, n):  # noqa: F811
    """the scratch of a product with Q8_0 weights (two rows and more a tile): one product's rows, quantized"""
    T = uninit
    w = fake(T, T.Q8_0_SPLIT, (4096, 1024), 1)
    x, y = rows(T, ne, nb), fake(T, T.F32, ne[::-1] + (4096,), 4)
    P = ctypes.POINTER(T.TskTensor)
    need = ctypes.c_size_t()
    assert T.load().tsk_workspace_size(T.OP_MUL_MAT, (P * 2)(ctypes.pointer(w), ctypes.pointer(x)), 2, ctypes.byref(y),
                                       ctypes.byref(need)) == 0
    # (up to four evenly spaced rows take none)
    evenly = n == ne[0] * ne[1] * ne[2]
    assert need.value == (0 if evenly and n <= 4 else (n * 1024 + 4 * n * 32 + 255) // 256 * 256)


@pytest.mark.parametrize("ne,nb,n", LAYOUTS)
def test_q8_0_quantize(uninit, ne, nb, n):  # noqa: F811
    T = uninit
    q = fake(T, T.Q8_0, ne[::-1] + (32,), 34)
    q.ne[0], q.nb[1] = 1024, 34 * 32
    q.nb[2], q.nb[3] = q.nb[1] * ne[0], q.nb[1] * ne[0] * ne[1]
    rc = T.load().tsk_q8_0_quantize(ctypes.byref(rows(T, ne, nb)), ctypes.byref(q), None)
    assert rc == (NOT_INIT if n == ne[0] * ne[1] * ne[2] else STRIDE)
