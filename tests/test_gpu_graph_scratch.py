"""Graphs whose calls take scratch from their stream's workspace: the buffer of the capture outlives the growth that later calls
bring, and a buffer bound in its place."""
import numpy as np
import pytest

from test_gpu_cross_attention import to
from test_gpu_int8 import T, dev, planes  # noqa: F401  (T: fixture)

pytestmark = pytest.mark.gpu


def states(T, rng, n, heads=2, d=64):  # noqa: F811
    return [to(T, rng.standard_normal((1, heads, n, d)), "bf16")[0] for _ in range(2)]


def replay(T, g, st, out, want):  # noqa: F811
    for _ in range(3):
        T._hipcheck(T.hip().hipMemset(out.ptr, 255, out.nbytes), "hipMemset")
        T.synchronize()
        g.launch()
        st.synchronize()
        assert np.array_equal(out.numpy(), want)


def test_growth_after_the_capture(T):  # noqa: F811
    """attention of few tokens (sums of ranges), then calls of more tokens and states, whose scratch is larger, and arrays where the
    first buffer would have been"""
    rng = np.random.default_rng(1)
    k, v = states(T, rng, 3000)
    q = to(T, rng.standard_normal((1, 2, 1, 64)), "bf16")[0]
    st, out = T.Stream(), T.empty((1, 1, 2, 64))
    assert T.workspace_size(T.OP_CROSS_ATTENTION, [q, k, v], out) > 0
    T.cross_attention(q, k, v, out=out, stream=st)
    st.synchronize()
    want = out.numpy()
    g = T.Graph(st, lambda: T.cross_attention(q, k, v, out=out, stream=st))
    held = []
    for n in (40, 700, 3000):
        q2, (k2, v2) = to(T, rng.standard_normal((1, 8, n, 128)), "bf16")[0], states(T, rng, 3000, 8, 128)
        out2 = T.empty((1, n, 8, 128))
        T.cross_attention(q2, k2, v2, out=out2, stream=st)
        W = T.i8_quantize(dev(T, rng.standard_normal((64, 2048)).astype(np.float32)))
        T.mul_mat(W, dev(T, np.ones((n * 200, 2048), np.float32)), stream=st)
        st.synchronize()
        held += [T.to_device(np.full((1 << 18,), np.nan, np.float32)) for _ in range(8)]
        replay(T, g, st, out, want)
    for h in held:
        assert np.isnan(h.numpy()).all()
    g.destroy()
    T.release_workspace(st)
    st.destroy()


def test_a_buffer_bound_after_the_capture(T):  # noqa: F811
    """an 8-bit product whose activations are quantized into scratch"""
    rng = np.random.default_rng(2)
    W, x = T.i8_quantize(dev(T, rng.standard_normal((96, 512)).astype(np.float32))), dev(T, rng.standard_normal((300, 512)).astype(np.float32))
    st, out = T.Stream(), T.empty((300, 96))
    T.mul_mat(W, x, out=out, stream=st)
    st.synchronize()
    want = out.numpy()
    g = T.Graph(st, lambda: T.mul_mat(W, x, out=out, stream=st))
    ws = T.empty((1 << 22,), "u8")
    T.set_workspace(ws, stream=st)
    replay(T, g, st, out, want)
    T.mul_mat(W, x, out=out, stream=st)
    st.synchronize()
    assert np.array_equal(out.numpy(), want)
    T.set_workspace(None, stream=st)
    replay(T, g, st, out, want)
    g.destroy()
    T.release_workspace(st)
    st.destroy()
