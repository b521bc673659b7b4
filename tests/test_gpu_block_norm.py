"""tsk_block_norm on gfx950 against 64 bits.

Tolerances. u = 2^-24. A sum over C values takes C / 256 additions per thread and
a tree of ten more at most: relative error (C / 256 + 12) u =: d u of the sum of
magnitudes. Mean and inverse deviation carry d u and (d / 2 + 3) u; a normalized
value (v - mean) inv w is then off by at most (d + 8) u of itself plus d u times
mean |v| inv |w|. Every further operation adds u of its result. The second norm is compared on the
residual as the kernel stored it (a bf16 tie decided the other way is no error of
the norm); a bf16 output adds 2^-8 of its value."""
import ctypes

import numpy as np
import pytest

import mxref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def T():
    from __graft_entry__ import ensure_built, load_tsk
    ensure_built()
    t = load_tsk()
    t.init(0)
    return t


def dev(T, x, dtype="f32"):
    return T.to_device(x) if dtype == "f32" else T.bf16_to_device(mxref.bf16_bits(x))


def host(a):
    return mxref.bf16_values(a.numpy()) if a.dtype == "bf16" else a.numpy()


def rounded(x, dtype):
    return x if dtype == "f32" else mxref.bf16_values(mxref.bf16_bits(x))


def norm_and_bound(v, kind, eps, w):
    """norm(v) * w in 64 bits and its error's bound"""
    c = v.shape[-1]
    d = c / 256 + 12
    n = mxref.norm(v, kind, eps) * w
    if kind == 0:
        return n, U * np.abs(n)
    dv = v - v.mean(-1, keepdims=True) if kind == 1 else v
    inv = 1 / np.sqrt((dv * dv).mean(-1, keepdims=True) + eps)
    b = (d + 8) * U * np.abs(n)
    if kind == 1:
        b = b + d * U * np.abs(v).mean(-1, keepdims=True) * inv * np.abs(w)
    return n, b


def make(rng, shape, dtype, mod, post_w, pre_w):
    B, S, C = shape
    f = lambda *s, std=1.0, add=0.0: (rng.standard_normal(s) * std + add).astype(np.float32)
    d = {"x": rounded(f(B, S, C, std=2.0, add=0.5), dtype), "y": rounded(f(B, S, C), dtype), "gate": None, "scale": None, "shift": None}
    if mod:
        n = {"c": (C,), "batch": (B, 1, C), "token": (B, S, C), "seq": (1, S, C)}[mod]
        d.update(gate=f(*n, std=0.5), scale=f(*n, std=0.3), shift=f(*n, std=0.3))
    d["post_w"] = f(C, std=0.1, add=1.0) if post_w else None
    d["pre_w"] = f(C, std=0.1, add=1.0) if pre_w else None
    return d


def check(T, d, dtype, post, pre, out_dtype, res_scale=1.0, in_place=False, eps=1e-5):
    up = lambda k: None if d[k] is None else T.to_device(d[k])
    x, y = dev(T, d["x"], dtype), dev(T, d["y"], dtype) if d["y"] is not None else None
    res = x if in_place else dev(T, np.full(d["x"].shape, 9.0, np.float32), dtype)
    dst = dev(T, np.full(d["x"].shape, 9.0, np.float32), out_dtype)
    keep = {k: up(k) for k in ("gate", "post_w", "pre_w", "scale", "shift")}
    T.block_norm(x, y, gate=keep["gate"], post=post, post_w=keep["post_w"], post_eps=eps, res_scale=res_scale, pre=pre,
                 pre_w=keep["pre_w"], pre_eps=eps, scale=keep["scale"], shift=keep["shift"], res=res, dst=dst)
    e = {k: None if v is None else v.astype(np.float64) for k, v in d.items()}
    r, br = res_scale * e["x"], 2 * U * np.abs(res_scale * e["x"])
    if y is not None:
        b, bb = norm_and_bound(e["y"], post, eps, 1.0 if e["post_w"] is None else e["post_w"])
        g = 1.0 if e["gate"] is None else e["gate"]
        r, br = r + g * b, br + np.abs(g) * (bb + 2 * U * np.abs(b))
    got_r = host(res).astype(np.float64)
    assert (np.abs(got_r - r) <= br + U * np.abs(r) + (2.0 ** -8 * np.abs(r) if dtype == "bf16" else 0)).all()
    h, bh = norm_and_bound(got_r, pre, eps, 1.0 if e["pre_w"] is None else e["pre_w"])
    if e["scale"] is not None:
        h, bh = h * (1 + e["scale"]), bh * np.abs(1 + e["scale"]) + 3 * U * np.abs(h) * (1 + np.abs(e["scale"]))
    if e["shift"] is not None:
        h = h + e["shift"]
    bh = bh + 2 * U * np.abs(h) + (2.0 ** -8 * np.abs(h) if out_dtype == "bf16" else 0)
    assert (np.abs(host(dst) - h) <= bh).all()
    return got_r, host(dst)


SHAPES = [(1, 1, 1), (2, 3, 16), (1, 5, 33), (2, 7, 63), (3, 1, 64), (2, 9, 77), (1, 4, 252), (2, 5, 256), (1, 3, 1000), (2, 194, 1024),
          (1, 3, 1028), (1, 2, 2048), (2, 3, 2816), (1, 2, 4096), (1, 2, 4099), (1, 2, 5120), (1, 3, 8192), (1, 2, 12292), (1, 2, 20000)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sizes(T, shape, dtype):
    rng = np.random.default_rng(sum(shape))
    check(T, make(rng, shape, dtype, "batch", True, True), dtype, T.NORM_RMS, T.NORM_LAYER, dtype)


@pytest.mark.parametrize("post", [0, 1, 2])
@pytest.mark.parametrize("pre", [0, 1, 2])
@pytest.mark.parametrize("mod", [None, "c", "batch", "token", "seq"])
def test_kinds_and_broadcasts(T, post, pre, mod):
    rng = np.random.default_rng(post * 3 + pre)
    d = make(rng, (3, 6, 96), "f32", mod, post > 0, pre == 2)
    check(T, d, "f32", post, pre, "bf16" if pre == 2 else "f32", res_scale=0.75 if post else 1.0, in_place=mod == "c")


@pytest.mark.parametrize("dtype,out", [("f32", "bf16"), ("bf16", "f32")])
def test_mixed_types(T, dtype, out):
    rng = np.random.default_rng(4)
    for c in (100, 1024, 2052):
        check(T, make(rng, (2, 11, c), dtype, "token", False, True), dtype, T.NORM_NONE, T.NORM_RMS, out)


def test_y_in_the_other_type(T):
    rng = np.random.default_rng(6)
    d = make(rng, (2, 5, 512), "f32", "batch", True, False)
    d["y"] = rounded(d["y"], "bf16")
    x, y, res = T.to_device(d["x"]), dev(T, d["y"], "bf16"), T.to_device(np.zeros_like(d["x"]))
    keep = [T.to_device(d["gate"]), T.to_device(d["post_w"])]
    T.block_norm(x, y, gate=keep[0], post=T.NORM_RMS, post_w=keep[1], pre=T.NORM_NONE, res=res)
    b, bb = norm_and_bound(d["y"].astype(np.float64), 2, 1e-5, d["post_w"].astype(np.float64))
    r = d["x"].astype(np.float64) + d["gate"].astype(np.float64) * b
    assert (np.abs(res.numpy() - r) <= np.abs(d["gate"]) * (bb + 2 * U * np.abs(b)) + 3 * U * np.abs(r) + 2 * U * np.abs(d["x"])).all()


@pytest.mark.parametrize("c", [1, 40, 1024, 5000])
def test_parts(T, c):
    """no branch, no residual output, the residual alone: the bits of the whole"""
    rng = np.random.default_rng(c)
    d = make(rng, (2, 13, c), "bf16", "batch", False, True)
    r, h = check(T, d, "bf16", T.NORM_NONE, T.NORM_LAYER, "f32")
    up = lambda k: T.to_device(d[k])
    x, y, w, g, sc, sh = dev(T, d["x"], "bf16"), dev(T, d["y"], "bf16"), up("pre_w"), up("gate"), up("scale"), up("shift")
    dst = T.empty(d["x"].shape)
    T.block_norm(x, y, gate=g, pre=T.NORM_LAYER, pre_w=w, scale=sc, shift=sh, dst=dst)
    assert np.array_equal(dst.numpy(), h)
    res = T.empty(d["x"].shape, "bf16")
    T.block_norm(x, y, gate=g, pre=T.NORM_NONE, res=res)
    assert np.array_equal(host(res), r)
    dst2 = T.empty(d["x"].shape)
    T.block_norm(res, pre=T.NORM_LAYER, pre_w=w, scale=sc, shift=sh, dst=dst2)
    assert np.array_equal(dst2.numpy(), h)
    d["y"] = None
    d["gate"] = None
    check(T, d, "bf16", T.NORM_NONE, T.NORM_RMS, "bf16", res_scale=1.5)


@pytest.mark.parametrize("c", [32, 96, 1024, 2816, 4096, 8224])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_mxfp4_output(T, c, dtype):
    """the bits of quantizing the f32 output"""
    rng = np.random.default_rng(c)
    d = make(rng, (2, 9, c), dtype, "token", True, False)
    d["x"][1, 3, 0] = np.nan                                   # a row of NaN: every block of it, no other
    up = lambda k: T.to_device(d[k])
    x, y, keep = dev(T, d["x"], dtype), dev(T, d["y"], dtype), [up(k) for k in ("gate", "post_w", "scale", "shift")]
    q = T.SplitMXFP4(T.empty((T.load().tsk_mxfp4_split_nbytes(c, 18),), "u8"), c, 18)
    f = T.empty(d["x"].shape)
    for dst in (q, f):
        T.block_norm(x, y, gate=keep[0], post=T.NORM_RMS, post_w=keep[1], pre=T.NORM_LAYER, scale=keep[2], shift=keep[3], dst=dst)
    codes, byte = mxref.quantize(f.numpy().reshape(18, c))
    assert np.array_equal(q.buf.numpy(), mxref.planes(codes, byte))
    assert (byte[12] == 255).all() and (np.delete(byte, 12, 0) != 255).all()


def test_strides(T):
    """rows with gaps, starts aligned to elements, outputs beside each other in one array; the rest stays"""
    rng = np.random.default_rng(8)
    B, S, C = 2, 5, 60
    wide = rng.standard_normal((B, S + 1, 3 * C + 5)).astype(np.float32)
    a = T.to_device(wide)
    ld = 3 * C + 5
    v = lambda off: a.view(off, (B, S, C), ((S + 1) * ld, ld, 1))
    x, y, res = v(1), v(1 + C), v(1 + 2 * C)
    g = rng.standard_normal((B, 1, C + 3)).astype(np.float32)
    gd = T.to_device(g)
    gate = gd.view(3, (B, 1, C), (C + 3, C + 3, 1))
    dst = T.empty((B, S, C))
    T.block_norm(x, y, gate=gate, pre=T.NORM_LAYER, res=res, dst=dst)
    after = a.numpy()
    cols = np.zeros(ld, bool)
    cols[1 + 2 * C:1 + 3 * C] = True
    r = wide[:, :S, 1:1 + C].astype(np.float64) + g[:, :, 3:].astype(np.float64) * wide[:, :S, 1 + C:1 + 2 * C]
    assert np.abs(after[:, :S][:, :, cols] - r).max() <= 2.0 ** -22 * np.abs(r).max()
    assert np.array_equal(after[:, :, ~cols], wide[:, :, ~cols]) and np.array_equal(after[:, S], wide[:, S])
    h, bh = norm_and_bound(after[:, :S][:, :, cols].astype(np.float64), 1, 1e-5, 1.0)
    assert (np.abs(dst.numpy() - h) <= bh + 2 * U * np.abs(h)).all()


@pytest.mark.parametrize("kind", [1, 2])
def test_ends(T, kind):
    """constant and zero rows, large means, rows of tiny and huge values"""
    c = 1024
    x = np.zeros((1, 5, c), np.float32)
    x[0, 1] = 3.0
    rng = np.random.default_rng(1)
    x[0, 2] = 1000.0 + rng.standard_normal(c)
    x[0, 3] = rng.standard_normal(c) * 1e-12
    x[0, 4] = rng.standard_normal(c) * 1e15
    dst = T.empty(x.shape)
    T.block_norm(T.to_device(x), pre=kind, pre_eps=1e-6, dst=dst)
    h, bh = norm_and_bound(x.astype(np.float64), kind, 1e-6, 1.0)
    got = dst.numpy()
    assert (got[0, 0] == 0).all() and np.isfinite(got).all()
    assert (np.abs(got - h) <= bh + 2 * U * np.abs(h)).all()


def test_stream_and_graph(T):
    """replayed on its own stream between eager work: the bits of the eager call"""
    rng = np.random.default_rng(2)
    d = make(rng, (2, 40, 1024), "f32", "batch", True, True)
    xs = [rng.standard_normal(d["x"].shape).astype(np.float32) for _ in range(3)]
    keep = {k: T.to_device(d[k]) for k in ("y", "gate", "post_w", "pre_w", "scale", "shift")}

    def run(x, res, dst, stream=None):
        T.block_norm(x, keep["y"], gate=keep["gate"], post=T.NORM_RMS, post_w=keep["post_w"], pre=T.NORM_LAYER, pre_w=keep["pre_w"],
                     scale=keep["scale"], shift=keep["shift"], res=res, dst=dst, stream=stream)
        return res, dst

    want = [[a.numpy() for a in run(T.to_device(x), T.empty(x.shape), T.empty(x.shape))] for x in xs]
    st = T.Stream()
    x, res, dst = T.to_device(xs[0]), T.empty(xs[0].shape), T.empty(xs[0].shape)
    T.synchronize()
    g = T.Graph(st, lambda: run(x, res, dst, st))
    for i in (0, 1, 2, 1):
        src = T.to_device(xs[i])
        T._hipcheck(T.hip().hipMemcpy(ctypes.c_void_p(x.ptr), ctypes.c_void_p(src.ptr), x.nbytes, 3), "hipMemcpy D2D")
        run(src, T.empty(xs[0].shape), T.empty(xs[0].shape))
        T.synchronize()
        g.launch()
        st.synchronize()
        assert np.array_equal(res.numpy(), want[i][0]) and np.array_equal(dst.numpy(), want[i][1])
    g.destroy()
    st.destroy()


def test_mlp_of_a_block(T):
    """the operators as a block uses them: gate and residual of the attention, norm and modulation into 4 bits, the
    4-bit projections of the MLP around its SwiGLU, then the MLP's own gate and residual. Each step in 64 bits from the
    step before as the kernels left it."""
    rng = np.random.default_rng(10)
    B, S, C, H = 2, 97, 256, 352
    d = make(rng, (B, S, C), "f32", "batch", False, False)
    n = B * S
    mats = [mxref.quantize((rng.standard_normal(s) * s[1] ** -0.5).astype(np.float32)) for s in ((H, C), (H, C), (C, H))]
    w1, w3, w2 = (T.SplitMXFP4(T.to_device(mxref.planes(*q)), q[0].shape[1], q[0].shape[0]) for q in mats)
    v1, v3, v2 = (mxref.values(*q) for q in mats)
    up = {k: T.to_device(d[k]) for k in ("x", "y", "gate", "scale", "shift")}
    h = T.SplitMXFP4(T.empty((T.load().tsk_mxfp4_split_nbytes(C, n),), "u8"), C, n)
    T.block_norm(up["x"], up["y"], gate=up["gate"], pre=T.NORM_LAYER, scale=up["scale"], shift=up["shift"], res=up["x"], dst=h)
    a, b = T.mul_mat(w1, h), T.mul_mat(w3, h)
    g = T.swiglu(a, b)
    q = T.mxfp4_quantize(g)
    o = T.mul_mat(w2, q)
    out = T.empty((B, S, C))
    T.block_norm(up["x"], o.view(0, (B, S, C), (S * C, C, 1)), gate=up["gate"], pre=T.NORM_NONE, res=out)
    f64 = lambda t: t.numpy().astype(np.float64)
    hv = mxref.values(*mxref.unplanes(h.buf.numpy(), n, C))
    r = d["x"].astype(np.float64) + d["gate"] * d["y"].astype(np.float64)
    x1 = f64(up["x"])
    assert np.abs(x1 - r).max() <= 4 * U * (np.abs(d["x"]) + np.abs(d["gate"] * d["y"])).max()
    m64 = mxref.norm(x1, 1, 1e-5) * (1 + d["scale"].astype(np.float64)) + d["shift"]
    # a code is at most half a step of its block from the value: 2^(e + 2) is at most amax, the widest step 2^(e + 1), saturation 2^(e + 1)
    amax = np.abs(m64).reshape(n, C // 32, 32).max(-1).repeat(32, -1)
    assert (np.abs(hv - m64.reshape(n, C)) <= amax * (0.5 + 2.0 ** -12)).all()
    for got, v in ((a, v1), (b, v3)):
        assert (np.abs(f64(got) - hv @ v.T) <= (C + 1) * 2.0 ** -23 * (np.abs(hv) @ np.abs(v).T)).all()
    codes, byte = mxref.quantize(g.numpy())
    assert np.array_equal(q.buf.numpy(), mxref.planes(codes, byte))
    qv = mxref.values(codes, byte)
    assert (np.abs(f64(o) - qv @ v2.T) <= (H + 1) * 2.0 ** -23 * (np.abs(qv) @ np.abs(v2).T)).all()
    want = x1 + d["gate"].astype(np.float64) * f64(o).reshape(B, S, C)
    assert (np.abs(f64(out) - want) <= 3 * U * (np.abs(x1) + np.abs(d["gate"]) * np.abs(f64(o).reshape(B, S, C)))).all()
