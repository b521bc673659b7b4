"""tsk_block_norm operation by operation: every product and sum is rounded for itself (but the two multiply-adds of a gate
and of a shift), in every kernel alike, so that the second norm reads the residual that is stored, whatever is asked for
beside it. All comparisons are of bits, on f32 rows, where nothing else rounds in between. Sizes: vectors of 8 in one
wave and in several, single values, rows longer than the registers hold."""
import numpy as np
import pytest

from test_gpu_block_norm import T  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu
SIZES = [64, 1000, 1024, 4096, 16384, 77, 1001, 5001, 16640, 20001]


def rows(rng, c, std=1.0, add=0.0):
    return (rng.standard_normal((7, c)) * std + add).astype(np.float32)


@pytest.mark.parametrize("c", SIZES)
def test_residual(T, c):
    """res_scale x + y in f32: a product, then a sum; with a weight of the branch's norm another product"""
    rng = np.random.default_rng(c)
    x, y, w, s = rows(rng, c, 2.0, 0.5), rows(rng, c), rows(rng, c)[0], np.float32(0.3)
    xd, yd, wd, res = T.to_device(x), T.to_device(y), T.to_device(w), T.empty(x.shape)
    T.block_norm(xd, yd, res_scale=float(s), pre=T.NORM_NONE, res=res)
    assert np.array_equal(res.numpy(), s * x + y)
    T.block_norm(xd, yd, post_w=wd, res_scale=float(s), pre=T.NORM_NONE, res=res)
    assert np.array_equal(res.numpy(), s * x + y * w)
    T.block_norm(xd, res_scale=float(s), pre=T.NORM_NONE, res=res)
    assert np.array_equal(res.numpy(), s * x)


@pytest.mark.parametrize("c", SIZES)
def test_modulation(T, c):
    """pre_w (1 + scale) x without norms: a product, a sum, a product"""
    rng = np.random.default_rng(c)
    x, w, sc, dst = rows(rng, c), rows(rng, c)[0], rows(rng, c, 0.3), T.empty((7, c))
    T.block_norm(T.to_device(x), pre=T.NORM_NONE, pre_w=T.to_device(w), scale=T.to_device(sc), dst=dst)
    assert np.array_equal(dst.numpy(), (x * w) * (np.float32(1) + sc))


@pytest.mark.parametrize("c", SIZES)
@pytest.mark.parametrize("pre", [1, 2])
def test_second_norm_reads_the_residual(T, c, pre):
    """the output in one call, without the residual, and from the residual of a call of its own"""
    rng = np.random.default_rng(c)
    xd, yd = T.to_device(rows(rng, c, 2.0, 0.5)), T.to_device(rows(rng, c))
    w, g, sc, sh = (T.to_device(v) for v in (rows(rng, c)[0], rows(rng, c), rows(rng, c), rows(rng, c)))
    whole, alone, after, res, res2 = (T.empty((7, c)) for _ in range(5))
    for branch in ({}, {"y": yd}, {"y": yd, "gate": g}, {"y": yd, "post": T.NORM_LAYER, "post_w": w},
                   {"y": yd, "post": T.NORM_RMS, "post_w": w, "gate": g}):
        branch["res_scale"] = 0.3
        for mod in ({}, {"pre_w": w}, {"scale": sc, "shift": sh}, {"pre_w": w, "scale": sc, "shift": sh}):
            T.block_norm(xd, pre=pre, res=res, dst=whole, **branch, **mod)
            T.block_norm(xd, pre=pre, dst=alone, **branch, **mod)
            T.block_norm(xd, pre=T.NORM_NONE, res=res2, **branch)
            T.block_norm(res2, pre=pre, dst=after, **mod)
            assert np.array_equal(res.numpy(), res2.numpy()), (sorted(branch), sorted(mod))
            assert np.array_equal(whole.numpy(), alone.numpy()), (sorted(branch), sorted(mod))
            assert np.array_equal(whole.numpy(), after.numpy()), (sorted(branch), sorted(mod))
