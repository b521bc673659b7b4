"""Scratch of products of few rows with 8-bit weights: none where they are quantized inside the product (no GPU needed)."""
import ctypes

import pytest

from test_abi import fake, tsk, uninit  # noqa: F401  (fixtures)
from test_cross_ops_abi import i8


@pytest.mark.parametrize("n,k,m,inside", [(1, 256, 32768, True), (1, 256, 32784, False), (4, 1024, 32768, True), (4, 1024, 32784, False),
                                          (1, 2048, 152064, True), (1, 2040, 152064, False), (1, 8192, 152064, True), (2, 2048, 152064, False),
                                          (5, 64, 64, False), (1, 8200, 64, False)])
def test_scratch(uninit, n, k, m, inside):  # noqa: F811
    T = uninit
    P = ctypes.POINTER(T.TskTensor)
    arr, got = (P * 2)(ctypes.pointer(i8(T, m, k)), ctypes.pointer(fake(T, T.F32, (n, k), 4))), ctypes.c_size_t()
    assert T.load().tsk_workspace_size(T.OP_MUL_MAT, arr, 2, ctypes.byref(fake(T, T.F32, (n, m), 4)), ctypes.byref(got)) == 0
    assert got.value == (0 if inside else (n * ((k + 15) // 16 * 16 + 4) + 255) // 256 * 256)
