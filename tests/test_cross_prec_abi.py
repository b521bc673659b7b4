"""The precisions that cross attention takes (no GPU needed)."""
from test_abi import fake, tsk, uninit  # noqa: F401  (fixtures)
from test_cross_ops_abi import ARG, NOT_INIT, at, cross_params
from test_mxfp4_abi import call


def test_precisions(uninit):  # noqa: F811
    T = uninit
    q, k = at(fake(T, T.BF16, (1, 2, 5, 64), 2), 0x100000), at(fake(T, T.BF16, (1, 2, 9, 64), 2), 0x200000)
    y = at(fake(T, T.F32, (1, 5, 2, 64), 4), 0x300000)
    for prec, rc in ((T.PREC_DEFAULT, NOT_INIT), (T.PREC_F32, NOT_INIT), (1, ARG), (-1, ARG), (11, ARG)):
        assert call(T, "tsk_cross_attention", q, k, k, cross_params(T, prec=prec), y) == rc
