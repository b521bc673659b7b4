"""The limits of cross attention's operands that the header states (no GPU needed)."""
import pytest

from test_abi import fake, tsk, uninit  # noqa: F401  (fixtures)
from test_cross_ops_abi import ALIGN, ARG, NOT_INIT, SHAPE, STRIDE, at, cross_params
from test_mxfp4_abi import call


def go(T, B, H, G, Nq, states=9, D=64, edit=None):
    q, k = at(fake(T, T.BF16, (B, H, Nq, D), 2), 0x10000000), at(fake(T, T.BF16, (B, G, states, D), 2), 0x20000000)
    y = at(fake(T, T.F32, (B, Nq, H, D), 4), 0x1000000000000)
    if edit:
        edit(q, k, y)
    return call(T, "tsk_cross_attention", q, k, k, cross_params(T), y)


@pytest.mark.parametrize("B,H,G", [(1, 1, 1), (2, 8, 4), (1, 4, 1)])
def test_rows(uninit, B, H, G):  # noqa: F811
    """32-row groups of the heads that share a key and value head, of all of them: 2^22"""
    most = 2 ** 22 // (B * G) * 32 // (H // G)
    assert go(uninit, B, H, G, most) == NOT_INIT
    assert go(uninit, B, H, G, most + 1) == SHAPE


def test_strides_of_states(uninit):  # noqa: F811
    """at least a row, at most 2^24 bytes; a single state's says nothing, nor do those of shared heads and sequences"""
    def step(n):
        def edit(q, k, y):
            k.nb[1] = n
        return edit

    for n, rc in ((128, NOT_INIT), (1 << 24, NOT_INIT), (112, STRIDE), (0, STRIDE), ((1 << 24) + 16, STRIDE), (136, ALIGN)):
        assert go(uninit, 2, 4, 2, 5, edit=step(n)) == rc
    assert go(uninit, 2, 4, 2, 5, states=1, edit=step(0)) == NOT_INIT

    def shared(q, k, y):
        k.nb[2] = k.nb[3] = q.nb[1] = q.nb[2] = q.nb[3] = 0

    assert go(uninit, 2, 4, 2, 5, edit=shared) == NOT_INIT


def test_scale(uninit):  # noqa: F811
    """a scale whose product with log2 e is no fp32 number would make every logit infinite or NaN"""
    T = uninit
    q, k = at(fake(T, T.BF16, (1, 2, 5, 64), 2), 0x100000), at(fake(T, T.BF16, (1, 2, 9, 64), 2), 0x200000)
    y = at(fake(T, T.F32, (1, 5, 2, 64), 4), 0x300000)
    for scale, rc in ((1e-45, NOT_INIT), (1.7e38, NOT_INIT), (2.0 ** 127, ARG), (3.4e38, ARG), (float("inf"), ARG), (-1.0, ARG)):
        assert call(T, "tsk_cross_attention", q, k, k, cross_params(T, scale=scale), y) == rc
