"""Rotary positions of one token of nearly 2^31 heads, dealt to waves of which the last has fewer, and of very many sequences."""
import numpy as np
import pytest

import crossref
import mxref
from test_gpu_int8 import T  # noqa: F401  (fixture)
from test_gpu_mxfp4_ends import fetch
from test_gpu_rope_axes import check, tolerance

pytestmark = pytest.mark.gpu


def test_the_most_heads(T):  # noqa: F811
    heads, n = (1 << 31) - 256, 4096
    x = T.empty((1, 1, heads, 2), "bf16")
    T._hipcheck(T.hip().hipMemset(x.ptr, 0, x.nbytes), "hipMemset")
    v = mxref.bf16_bits(np.random.default_rng(1).standard_normal(2 * n).astype(np.float32))
    places = (0, (1 << 30) - 5, heads - (1 << 20) - 99, heads - n)        # (within the last wave's heads, and its last)
    for at in places:
        T._hipcheck(T.hip().hipMemcpy(x.ptr + 4 * at, v.ctypes.data, v.nbytes, 1), "hipMemcpy H2D")
    T.rope_axes(x, T.to_device(np.array([[2]], np.int32)), (2,), out=x)
    a = mxref.bf16_values(v).reshape(1, 1, n, 2)
    want, size = crossref.turn(a, np.full((1, 1, 1), 2), (2,), False, False)
    for at in places:
        got = mxref.bf16_values(fetch(T, x, 4 * at, (2 * n,), np.uint16)).reshape(1, 1, n, 2)
        assert (np.abs(got - want) - tolerance(a, size, want, 2.0, False, "bf16")).max() <= 0, at


@pytest.mark.parametrize("b,s,h,d", [(9001, 1, 3, 32), (4096, 1, 16, 128), (700, 13, 2, 20), (3000, 4, 1, 64)])
@pytest.mark.parametrize("shared", [False, True])
def test_many_short_sequences(T, b, s, h, d, shared):  # noqa: F811
    """more sequences than waves, and fewer; positions of their own and one array for all"""
    rng = np.random.default_rng(b)
    x = rng.standard_normal((b, s, h, d)).astype(np.float32)
    pos = rng.integers(0, 3000, (1 if shared else b, 2, s)).astype(np.int32)
    check(T, x, pos, (d - 8, 8), w=(1 + 0.1 * rng.standard_normal(d)).astype(np.float32), dtype="bf16" if d == 128 else "f32")
