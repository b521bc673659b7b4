"""A block's cross attention from end to end on gfx950: norm and modulation into 8-bit rows, projections of the tokens and
of the states, positions of both over time, height and width, attention to the states that count, the projection back.

Every stage is held to the 64-bit result for what the stage before it left on the device, by the tolerances of its own
tests; the run as a whole is captured and replayed with other tokens, whose bits are those of an eager run."""
import ctypes

import numpy as np
import pytest

import crossref
import mxref
import test_gpu_cross_attention as attn
import test_gpu_rope_axes as rope
from test_gpu_int8 import T, dev, host, off, want_linear  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


class Block:
    def __init__(self, T, B, N, frames, h, w, c, heads, d, seed):  # noqa: F811
        rng = np.random.default_rng(seed)
        self.T, self.B, self.N, self.M, self.c, self.heads, self.d = T, B, N, frames * h * w, c, heads, d
        self.dims = (d // 2, d // 4, d // 4)
        hd = heads * d
        self.W = {n: crossref.i8_quantize(rng.standard_normal(s).astype(np.float32) / np.sqrt(s[1]))
                  for n, s in (("q", (hd, c)), ("kv", (2 * hd, c)), ("o", (c, hd)))}
        self.Wd = {n: T.SplitI8(T.to_device(crossref.i8_planes(*w)), w[0].shape[1], w[0].shape[0]) for n, w in self.W.items()}
        self.norm = [(1 + 0.1 * rng.standard_normal(d)).astype(np.float32) for _ in range(2)]
        self.normd = [T.to_device(w) for w in self.norm]
        self.bias = rng.standard_normal(c).astype(np.float32)
        t, y, x = np.meshgrid(np.arange(frames) * 2.7, np.arange(h), np.arange(w), indexing="ij")
        self.kpos = np.stack([t.ravel(), y.ravel(), x.ravel()]).astype(np.float32)
        self.qpos = np.stack([np.arange(N), np.zeros(N), np.zeros(N)]).astype(np.float32)
        self.lens = np.array([self.M, self.M // 2] + [0] * (B - 2), np.int32)[:B]
        self.states = mxref.bf16_values(mxref.bf16_bits(rng.standard_normal((B * self.M, c)).astype(np.float32)))
        self.mod = [rng.standard_normal((B, 1, c)).astype(np.float32) * 0.3 for _ in range(2)]
        self.scale, self.shift, self.statesd = T.to_device(self.mod[0]), T.to_device(self.mod[1]), dev(T, self.states, "bf16")
        self.pos = [T.to_device(self.qpos), T.to_device(self.kpos)]
        self.lend, self.biasd = T.to_device(self.lens), T.to_device(self.bias)
        self.x = T.empty((B, N, c))
        self.h = T.i8_quantize(T.to_device(np.zeros((B * N, c), np.float32)))
        self.q0, self.q1 = T.empty((B, N, heads, d), "bf16"), T.empty((B, N, heads, d), "bf16")
        self.kv0, self.k1 = T.empty((B, self.M, 2, heads, d), "bf16"), T.empty((B, self.M, heads, d), "bf16")
        self.o, self.out = T.empty((B, N, heads, d), "bf16"), T.empty((B, N, c))

    def run(self, stream=None):
        T, B, N, M, H, d = self.T, self.B, self.N, self.M, self.heads, self.d
        hd = H * d
        T.block_norm(self.x, pre=T.NORM_LAYER, scale=self.scale, shift=self.shift, dst=self.h, stream=stream)
        T.mul_mat(self.Wd["q"], self.h, out=self.q0.view(0, (B * N, hd), (hd, 1)), stream=stream)
        T.mul_mat(self.Wd["kv"], self.statesd, out=self.kv0.view(0, (B * M, 2 * hd), (2 * hd, 1)), stream=stream)
        T.rope_axes(self.q0, self.pos[0], self.dims, w=self.normd[0], out=self.q1, stream=stream)
        k = self.kv0.view(0, (B, M, H, d), (M * 2 * hd, 2 * hd, d, 1))
        T.rope_axes(k, self.pos[1], self.dims, w=self.normd[1], out=self.k1, stream=stream)
        heads = lambda t, n: t.view(0, (B, H, n, d), (n * hd, d, hd, 1))
        v = self.kv0.view(hd, (B, H, M, d), (M * 2 * hd, d, 2 * hd, 1))
        T.cross_attention(heads(self.q1, N), heads(self.k1, M), v, kv_len=self.lend, out=self.o, stream=stream)
        T.mul_mat(self.Wd["o"], self.o.view(0, (B * N, hd), (hd, 1)), bias=self.biasd, out=self.out.view(0, (B * N, self.c), (self.c, 1)),
                  stream=stream)

    def put(self, x):
        src = self.T.to_device(x)
        self.T._hipcheck(self.T.hip().hipMemcpy(ctypes.c_void_p(self.x.ptr), ctypes.c_void_p(src.ptr), src.nbytes, 3), "hipMemcpy D2D")


@pytest.mark.parametrize("B,N,frames,h,w,c,heads,d", [(2, 194, 16, 4, 4, 256, 4, 64), (1, 1, 64, 3, 5, 128, 2, 128), (3, 40, 5, 1, 7, 96, 3, 32)])
def test_block(T, B, N, frames, h, w, c, heads, d):  # noqa: F811
    blk = Block(T, B, N, frames, h, w, c, heads, d, N)
    rng = np.random.default_rng(c)
    xs = [(rng.standard_normal((B, N, c)) * 2 + 0.3).astype(np.float32) for _ in range(3)]
    hd, M = heads * d, blk.M
    want = []
    for x in xs:
        blk.put(x)
        blk.run()
        want.append(blk.out.numpy())
    # the last of them, stage by stage
    y = T.to_device(np.zeros((B, N, c), np.float32))
    T.block_norm(blk.x, pre=T.NORM_LAYER, scale=blk.scale, shift=blk.shift, dst=y)
    hq = crossref.i8_quantize(y.numpy().reshape(B * N, c))
    got = crossref.i8_unplanes(blk.h.buf.numpy(), B * N, c)
    assert np.array_equal(got[0][:, :c], hq[0]) and np.array_equal(got[1], hq[1])
    q0, q1, kv0, k1, o = (host(t) for t in (blk.q0, blk.q1, blk.kv0, blk.k1, blk.o))
    ref, tol = want_linear(hq, blk.W["q"], None, "bf16")
    assert off(q0.reshape(B * N, hd), ref, tol) <= 0
    ref, tol = want_linear(crossref.i8_quantize(blk.states), blk.W["kv"], None, "bf16")
    assert off(kv0.reshape(B * M, 2 * hd), ref, tol) <= 0
    for before, after, pos, nw in ((q0, q1, blk.qpos, blk.norm[0]), (kv0[:, :, 0], k1, blk.kpos, blk.norm[1])):
        r = crossref.rms(before, nw.astype(np.float64), np.float32(1e-6))
        ref, size = crossref.turn(r, pos[None], blk.dims, False, False)
        assert (np.abs(after - ref) - rope.tolerance(r, size, ref, np.abs(pos).max(), True, "bf16")).max() <= 0
    k, v = k1.transpose(0, 2, 1, 3), kv0[:, :, 1].transpose(0, 2, 1, 3)
    ref, size, big = crossref.attention(q1.transpose(0, 2, 1, 3), k, v, np.float32(d ** -0.5), np.arange(M) < blk.lens[:, None])
    assert (np.abs(o - ref) - attn.tolerance(ref, size, big, d, M, "bf16", "bf16", np.abs(v).max())).max() <= 0
    assert (o[blk.lens == 0] == 0).all()
    ref, tol = want_linear(crossref.i8_quantize(o.reshape(B * N, hd)), blk.W["o"], blk.bias, "f32")
    assert off(want[2].reshape(B * N, c), ref, tol) <= 0
    # as one graph
    st = T.Stream()
    T.synchronize()
    blk.run(st)                                                # (the stream's workspace exists before the capture)
    st.synchronize()
    assert np.array_equal(blk.out.numpy(), want[2])
    g = T.Graph(st, lambda: blk.run(st))
    for i in (0, 1, 2, 0):
        blk.put(xs[i])
        T.i8_quantize(blk.statesd)                             # eager work between the replays
        T.synchronize()
        g.launch()
        st.synchronize()
        assert np.array_equal(blk.out.numpy(), want[i])
    g.destroy()
    st.destroy()
