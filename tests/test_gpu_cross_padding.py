"""Cross attention: tokens from q_len on hold anything, and have no effect on the others."""
import numpy as np
import pytest

from test_gpu_cross_attention import host, shape, to  # noqa: F401  (shape: fixture)
from test_gpu_int8 import T  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,D", [("bf16", 64), ("bf16", 128), ("f16", 96)])
@pytest.mark.parametrize("rows,ranges", [(32, 1), (32, 4), (128, 1), (128, 4), (256, 1), (256, 4)])
def test_tokens_past_the_last_have_no_effect(T, shape, rows, ranges, kv, D):  # noqa: F811
    """the same bits whatever they hold; they stand in the same waves as tokens that count, of one head and of two that share a
    key and value head"""
    shape(rows, ranges)
    rng = np.random.default_rng(D)
    B, H, Nq, Nkv = 2, 2, 300, 1000
    q_len = np.array([201, 9], np.int32)
    q = rng.standard_normal((B, H, Nq, D)).astype(np.float32) * 3
    behind = np.broadcast_to((np.arange(Nq) >= q_len[:, None])[:, None, :, None], q.shape)
    for G in (2, 1):
        K, V = (to(T, rng.standard_normal((B, G, Nkv, D)), kv)[0] for _ in range(2))
        want = None
        for fill in (0.0, np.nan, np.inf, -np.inf, 6e4, -1e3):
            qt = "f32" if fill == 6e4 else kv
            out, _ = to(T, np.full((B, Nq, H, D), 77.0), "f32")
            Q = to(T, np.where(behind, np.float32(fill), to(T, q, kv)[1]), qt)[0]
            got = host(T.cross_attention(Q, K, V, q_len=T.to_device(q_len), out=out))
            left = np.arange(Nq) >= q_len[:, None]
            assert (got[left] == 77.0).all()
            want = got if want is None else want
            assert np.isfinite(got).all() and np.array_equal(got, want), (G, fill)
