"""Performance cases of the operators around cross attention to an encoder's
states: products in 8-bit integers with a scale for each token and channel,
rotary positions over several axes, and attention to states of another length.

With `own` the calls a user makes of libtsk.so, else the same operators in
elementary torch operations. 8-bit rows hold, for a row x, the scale d =
max(amax, 2^-100) / 127 as a float32 and the integers nearest to x / d, ties to
even; the planes are rows of K integers, padded with zeros to 16 bytes, then a
scale a row. Sizes are the models': 194 / 646 latent tokens of a 9 s /
30 s clip, batches of 2, hidden 1024 in 16 heads of 64, 77 text tokens, T5
2048 and 5120; and generic ones.
"""
import ctypes
import math

import torch

own = False
DEV = "cuda"
EPS = 1e-6
TINY = 2.0 ** -100


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # the activations of one 9 s clip on their way into an 8-bit product, and back: launch latency
        {"name": "quantize_9s", "kind": "quantize", "type": "f32", "rows": 388, "k": 1024},
        # a large weight matrix, once at load
        {"name": "quantize_weights", "kind": "quantize", "type": "bf16", "rows": 8192, "k": 8192},
        # adaLN of one conditioning row: a single token against 8-bit weights
        {"name": "linear_one_row", "kind": "linear", "act": "bf16", "rows": 1, "k": 1024, "m": 6144, "out": "f32", "bias": True},
        # a few rows against a large layer: the weights' bytes
        {"name": "linear_few_rows", "kind": "linear", "act": "bf16", "rows": 8, "k": 8192, "m": 8192, "out": "bf16", "bias": False},
        # T5's projection back to its width over several texts, ragged in rows and outputs
        {"name": "linear_ragged", "kind": "linear", "act": "bf16", "rows": 2047, "k": 5120, "m": 2050, "out": "bf16", "bias": True},
        # a large product of two 8-bit operands: the matrix unit's rate
        {"name": "linear_large", "kind": "linear", "act": "i8", "rows": 8192, "k": 8192, "m": 8192, "out": "bf16", "bias": False},
        # queries of a 9 s clip: norm of each head and two axes, time and channel group
        {"name": "rope_9s", "kind": "rope", "type": "f32", "batch": 2, "seq": 194, "heads": 16, "d": 64, "dims": "48,16",
         "pairs": "adjacent", "shared": False, "pos": "f32", "norm": True},
        # frames of 32 x 32 patches over time, height and width: memory
        {"name": "rope_video", "kind": "rope", "type": "bf16", "batch": 1, "seq": 16384, "heads": 16, "d": 128, "dims": "44,42,42",
         "pairs": "adjacent", "shared": False, "pos": "i32", "norm": False},
        # the latent tokens of a 30 s clip to its text, one of the two texts short
        {"name": "cross_text", "kind": "cross", "type": "bf16", "batch": 2, "nq": 646, "nkv": 77, "heads": 16, "kv_heads": 16, "d": 64,
         "mask": "len"},
        # one token a sequence to long states, four heads to a pair of key and value: the states' bytes
        {"name": "cross_one_query", "kind": "cross", "type": "bf16", "batch": 4, "nq": 1, "nkv": 16384, "heads": 32, "kv_heads": 8,
         "d": 128, "mask": "len"},
        # many tokens to the states of a long video: the matrix unit's rate
        {"name": "cross_long", "kind": "cross", "type": "bf16", "batch": 1, "nq": 4096, "nkv": 8192, "heads": 16, "kv_heads": 16,
         "d": 128, "mask": "none"},
        # from the residual stream of a 30 s clip to the attention's output: norm and modulation into 8 bits, projections of the tokens
        # and of the video's states, positions of both, attention
        {"name": "block_30s", "kind": "block", "batch": 2, "nq": 646, "frames": 64, "height": 4, "width": 4, "c": 1024, "heads": 16,
         "d": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "linear", "rope", "rope", "cross", "cross", "cross", "block"])
    if kind == "quantize":
        return {"kind": kind, "type": rng.choice(["f32", "bf16"]), "rows": _log(rng, 1, 8192), "k": _log(rng, 1, 8192)}
    if kind == "linear":
        act = rng.choice(["bf16", "f32", "i8", "i8"])
        k, m = _log(rng, 16, 8192), _log(rng, 16, 8192)
        return {"kind": kind, "act": act, "rows": _log(rng, 1, 8192), "k": k, "m": m, "out": rng.choice(["f32", "bf16"]),
                "bias": rng.random() < 0.5}
    if kind == "rope":
        n = rng.choice([1, 2, 3, 4])
        dims = [2 * rng.randint(1, 32) for _ in range(n)]
        case = {"kind": kind, "type": rng.choice(["f32", "bf16"]), "batch": rng.choice([1, 2, 4]), "seq": _log(rng, 1, 16384),
                "heads": _log(rng, 1, 32), "d": sum(dims) + rng.choice([0, 0, 0, 1, 8, 32]), "dims": ",".join(map(str, dims)),
                "pairs": rng.choice(["adjacent", "halves"]), "shared": rng.random() < 0.5, "pos": rng.choice(["i32", "f32"]),
                "norm": rng.random() < 0.5}
        case["seq"] = max(1, min(case["seq"], (1 << 25) // (case["batch"] * case["heads"] * case["d"])))
        return case
    if kind == "block":
        d = rng.choice([32, 64, 128])
        return {"kind": kind, "batch": rng.choice([1, 2, 4]), "nq": _log(rng, 1, 1024), "frames": _log(rng, 1, 64),
                "height": rng.randint(1, 5), "width": rng.randint(1, 5), "c": 16 * _log(rng, 4, 64), "heads": _log(rng, 1, 16), "d": d}
    kv, d = _log(rng, 1, 16), 8 * rng.choice([4, 5, 8, 8, 9, 12, 16, 16])
    case = {"kind": kind, "type": rng.choice(["bf16", "f16"]), "batch": rng.choice([1, 2, 3, 4]), "nq": _log(rng, 1, 4096),
            "nkv": _log(rng, 1, 16384), "heads": kv * rng.choice([1, 1, 2, 4]), "kv_heads": kv, "d": d,
            "mask": rng.choice(["none", "len", "len", "holes"])}
    most = 4096 * 8192 * 16 * 128
    case["nq"] = max(1, min(case["nq"], most // (case["batch"] * case["heads"] * case["nkv"] * d)))
    return case


# ---------------------------------------------------------------- inputs
class _Rand:
    """seeded inputs, made on the GPU"""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(1 + int(seed))

    def __call__(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.g, device=DEV, dtype=torch.float32) * std

    def whole(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device=DEV, dtype=torch.int32)


TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _padded(x):
    """rows whose strides are multiples of 16 bytes, as a view of x's columns"""
    per = 16 // x.element_size()
    y = torch.empty(*x.shape[:-1], (x.shape[-1] + per - 1) // per * per, dtype=x.dtype, device=DEV)[..., :x.shape[-1]]
    return y.copy_(x)


def _pack(q, d):
    """8-bit planes, one array of bytes"""
    rows, k = q.shape
    b = torch.zeros(rows, (k + 15) // 16 * 16, dtype=torch.int8, device=DEV)
    b[:, :k] = q
    return torch.cat([b.reshape(-1).view(torch.uint8), d.float().reshape(-1).view(torch.uint8)])


def _unpack(planes, rows, k):
    ld = (k + 15) // 16 * 16
    return planes[:rows * ld].view(torch.int8).reshape(rows, ld)[:, :k].float(), planes[rows * ld:].view(torch.float32)[:, None]


def _codes(x):
    """f32 rows: the integers, and the scale of each row; quotients next to a half need 64 bits, and torch takes a division by a
    plain number as a product with its inverse"""
    d = (x.abs().amax(-1, keepdim=True).clamp(min=TINY).double() / 127.0).float()
    return torch.round(x.double() / d).float(), d


def _weights(r, m, k):
    return _pack(*_codes(r(m, k, std=k ** -0.5) * torch.exp(r(m, 1, std=0.3))))


def _planes_for(rows, k):
    return torch.empty(rows * ((k + 15) // 16 * 16) + 4 * rows, dtype=torch.uint8, device=DEV)


def _dims(case):
    return [int(v) for v in case["dims"].split(",")]


def _lengths(case, r, b, n):
    """the states that count: all of the first sequence's, a part of the others'; often short, now and then none"""
    if case["mask"] != "len":
        return None
    v = r.whole(0, n + 1, b)
    v[0] = n
    return v


def _grid(f, h, w, rate):
    """the positions of f frames of h x w patches, their times on the clock of the tokens"""
    t, y, x = torch.meshgrid([torch.arange(n, device=DEV, dtype=torch.float32) for n in (f, h, w)], indexing="ij")
    return torch.stack([t.reshape(-1) * rate, y.reshape(-1), x.reshape(-1)])


def prepare(case, seed):
    r, kind, st = _Rand(seed), case["kind"], {"case": case}
    if kind == "quantize":
        n, k = case["rows"], case["k"]
        # rows of different sizes, as activations and weight rows have
        st["x"] = (r(n, k) * torch.exp(r(n, 1))).to(TYPES[case["type"]])
        st["planes"], st["out"] = _planes_for(n, k), torch.empty(n, k, device=DEV)
    elif kind == "linear":
        n, k, m = case["rows"], case["k"], case["m"]
        x = r(n, k) * torch.exp(r(n, 1, std=0.5))
        st["x"] = _pack(*_codes(x)) if case["act"] == "i8" else _padded(x.to(TYPES[case["act"]]))
        st["bias"] = r(m, std=0.02) if case["bias"] else None
        st["weights"] = _weights(r, m, k)
        st["out"] = _padded(torch.zeros(n, m, dtype=TYPES[case["out"]], device=DEV))
    elif kind == "rope":
        b, s, n = case["batch"], case["seq"], len(_dims(case))
        st["x"] = r(b, s, case["heads"], case["d"]).to(TYPES[case["type"]])
        st["w"] = 1 + r(case["d"], std=0.1) if case["norm"] else None
        st["pos"] = r.whole(0, 20000, b, n, s) if case["pos"] == "i32" else r(b, n, s).abs() * 500
        st["out"] = torch.empty_like(st["x"])
    elif kind == "cross":
        b, nq, nkv, d, typ = case["batch"], case["nq"], case["nkv"], case["d"], TYPES[case["type"]]
        # tokens and states as projections leave them: heads side by side
        st["q"] = r(b, nq, case["heads"], d).to(typ)
        st["k"] = r(b, nkv, case["kv_heads"], d).to(typ)
        st["v"] = r(b, nkv, case["kv_heads"], d).to(typ)
        st["len"] = _lengths(case, r, b, nkv)
        st["valid"] = (r.whole(0, 4, b, nkv) > 0).to(torch.uint8) if case["mask"] == "holes" else None
        st["out"] = torch.empty_like(st["q"])
    else:
        b, nq, c, h, d = case["batch"], case["nq"], case["c"], case["heads"], case["d"]
        f, y, x = case["frames"], case["height"], case["width"]
        n = f * y * x
        st.update(x=r(b, nq, c, std=2.0) + 0.3, scale=r(b, 1, c, std=0.3), shift=r(b, 1, c, std=0.3), states=r(b, n, c).bfloat16())
        st.update(wq=_weights(r, h * d, c), wkv=_weights(r, 2 * h * d, c), qw=1 + r(d, std=0.1), kw=1 + r(d, std=0.1))
        st["kpos"] = _grid(f, y, x, 2.7)
        st["qpos"] = torch.cat([torch.arange(nq, device=DEV).float()[None], torch.zeros(2, nq, device=DEV)])
        v = r.whole(1, f + 1, b) * (y * x)                    # whole frames
        v[0] = n
        st["len"] = v
        st.update(planes=_planes_for(b * nq, c), q=torch.empty(b, nq, h, d, dtype=torch.bfloat16, device=DEV),
                  kv=torch.empty(b, n, 2, h, d, dtype=torch.bfloat16, device=DEV),
                  out=torch.empty(b, nq, h, d, dtype=torch.bfloat16, device=DEV))
    return st


# ---------------------------------------------------------------- one pass
def _plain_linear(x, planes, m, bias):
    """x: integers and scales of the rows"""
    w, d = _unpack(planes, m, x[0].shape[1])
    y = (x[0] @ w.T) * x[1] * d.T
    return y if bias is None else y + bias


def _turns(dims, shared):
    """turns of each pair per position, and its axis"""
    n = sum(dims)
    axis = [a for a, k in enumerate(dims) for _ in range(k // 2)]
    own_pair = [j for k in dims for j in range(k // 2)]
    power = [2 * i / n if shared else 2 * j / dims[a] for i, (a, j) in enumerate(zip(axis, own_pair))]
    f = torch.tensor(power, dtype=torch.float64, device=DEV)
    return torch.exp2(-f * math.log2(10000.0)), torch.tensor(axis, device=DEV)


def _plain_rope(x, w, pos, dims, pairs, shared):
    """x (b, s, h, d) in f32; pos (b or 1, n, s)"""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    f, axis = _turns(dims, shared)
    # angles of far positions need 64 bits
    angle = pos.double()[:, axis].transpose(1, 2) * f
    c, s = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    n = sum(dims)
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if pairs == "adjacent" else (x[..., :n // 2], x[..., n // 2:n])
    u, v = a * c - b * s, a * s + b * c
    turned = torch.stack([u, v], -1).flatten(-2) if pairs == "adjacent" else torch.cat([u, v], -1)
    return torch.cat([turned, x[..., n:]], -1)


def _counts(st, nkv):
    """which states count, (b, nkv), or None"""
    if st.get("len") is not None:
        return torch.arange(nkv, device=DEV) < st["len"][:, None]
    return st["valid"] != 0 if st.get("valid") is not None else None


def _plain_cross(q, k, v, counts):
    """q (b, nq, h, d), k, v (b, nkv, g, d) in f32"""
    b, nq, h, d = q.shape
    g = k.shape[2]
    if counts is not None:
        v = torch.where(counts[:, :, None, None], v, 0.0)
    q = q.permute(0, 2, 1, 3).reshape(b, g, h // g * nq, d)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)) * d ** -0.5
    if counts is not None:
        s = s.masked_fill(~counts[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
    o = torch.matmul(p, v.permute(0, 2, 1, 3)) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.reshape(b, h, nq, d).permute(0, 2, 1, 3)


def _block_dims(d):
    return [d // 2, d // 4, d // 4]


def _plain(st):
    case = st["case"]
    if case["kind"] == "quantize":
        q, d = _codes(st["x"].float())
        return q * d
    if case["kind"] == "linear":
        x = _unpack(st["x"], case["rows"], case["k"]) if case["act"] == "i8" else _codes(st["x"].float())
        return _plain_linear(x, st["weights"], case["m"], st["bias"]).to(TYPES[case["out"]])
    if case["kind"] == "rope":
        return _plain_rope(st["x"].float(), st["w"], st["pos"], _dims(case), case["pairs"], case["shared"]).to(st["x"].dtype)
    if case["kind"] == "cross":
        return _plain_cross(st["q"].float(), st["k"].float(), st["v"].float(), _counts(st, case["nkv"])).to(st["q"].dtype)
    h, d = case["heads"], case["d"]
    x = st["x"] - st["x"].mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + st["scale"]) + st["shift"]
    q = _plain_linear(_codes(x.flatten(0, 1)), st["wq"], h * d, None).bfloat16().float().reshape(st["q"].shape)
    kv = _plain_linear(_codes(st["states"].float().flatten(0, 1)), st["wkv"], 2 * h * d, None).bfloat16().float().reshape(st["kv"].shape)
    q = _plain_rope(q, st["qw"], st["qpos"][None], _block_dims(d), "adjacent", False).bfloat16().float()
    k = _plain_rope(kv[:, :, 0], st["kw"], st["kpos"][None], _block_dims(d), "adjacent", False).bfloat16().float()
    o = _plain_cross(q, k, kv[:, :, 1], _counts(st, kv.shape[1]))
    return {"kv": torch.stack([k, kv[:, :, 1]], 2).bfloat16(), "out": o.bfloat16()}


def _plan(st):
    """the descriptors of the calls, built once for the buffers that the program keeps"""
    from __graft_entry__ import load_tsk
    t = load_tsk()
    t.init(0)
    types = {torch.float32: t.F32, torch.bfloat16: t.BF16, torch.float16: t.F16, torch.int32: t.I32}
    lib, case = t.load(), st["case"]

    def d(x):
        return None if x is None else ctypes.pointer(t.desc(x, types[x.dtype]))

    def planes(x, rows, k):
        return ctypes.pointer(t.desc(t.SplitI8(x, k, rows), t.I8_SPLIT))

    def rope(x, w, pos, dims, pairs, shared, out):
        p = t.RopeAxesParams()
        p.n_axes, p.freq_base, p.freq_scale, p.eps, p.w = len(dims), 10000.0, 1.0, EPS, d(w)
        for i, v in enumerate(dims):
            p.dims[i] = v
        p.pairs = t.ROPE_ADJACENT if pairs == "adjacent" else t.ROPE_HALVES
        p.shared_freqs = shared
        return lib.tsk_rope_axes, (d(x), d(pos), ctypes.pointer(p), d(out))

    def cross(q, k, v, out):
        p = t.CrossAttnParams()
        p.scale, p.kv_len = q.shape[-1] ** -0.5, d(st.get("len"))
        if st.get("valid") is not None:
            p.kv_valid, p.kv_valid_nb = st["valid"].data_ptr(), st["valid"].stride(0)
        q, k, v = (x.permute(0, 2, 1, 3) for x in (q, k, v))
        return lib.tsk_cross_attention, (d(q), d(k), d(v), ctypes.pointer(p), d(out))

    if case["kind"] == "quantize":
        q = planes(st["planes"], case["rows"], case["k"])
        return t.check, [(lib.tsk_i8_quantize, (d(st["x"]), q)), (lib.tsk_i8_dequantize, (q, d(st["out"])))]
    if case["kind"] == "linear":
        n, k, m = case["rows"], case["k"], case["m"]
        x = planes(st["x"], n, k) if case["act"] == "i8" else d(st["x"])
        return t.check, [(lib.tsk_mul_mat, (planes(st["weights"], m, k), x, d(st["bias"]), d(st["out"])))]
    if case["kind"] == "rope":
        return t.check, [rope(st["x"], st["w"], st["pos"], _dims(case), case["pairs"], case["shared"], st["out"])]
    if case["kind"] == "cross":
        return t.check, [cross(st["q"], st["k"], st["v"], st["out"])]
    b, nq, c, n, hd = case["batch"], case["nq"], case["c"], st["kv"].shape[1], case["heads"] * case["d"]
    p = t.BlockNormParams()
    p.res_scale, p.pre_norm, p.pre_eps, p.scale, p.shift = 1.0, t.NORM_LAYER, EPS, d(st["scale"]), d(st["shift"])
    h = planes(st["planes"], b * nq, c)                       # [c, nq, b] for the norm, [c, b nq] for the product: the same rows
    h3 = planes(st["planes"], b * nq, c)
    h3.contents.ne[1], h3.contents.ne[2] = nq, b
    dims = _block_dims(case["d"])
    k, v = st["kv"][:, :, 0], st["kv"][:, :, 1]
    return t.check, [(lib.tsk_block_norm, (d(st["x"]), None, ctypes.pointer(p), None, h3)),
                     (lib.tsk_mul_mat, (planes(st["wq"], hd, c), h, None, d(st["q"].view(b * nq, hd)))),
                     (lib.tsk_mul_mat, (planes(st["wkv"], 2 * hd, c), d(st["states"].view(b * n, c)), None,
                                        d(st["kv"].view(b * n, 2 * hd)))),
                     rope(st["q"], st["qw"], st["qpos"], dims, "adjacent", False, st["q"]),
                     rope(k, st["kw"], st["kpos"], dims, "adjacent", False, k),
                     cross(st["q"], k, v, st["out"])]


def _own(st):
    if "plan" not in st:
        st["plan"] = _plan(st)
    check, calls = st["plan"]
    stream = torch.cuda.current_stream().cuda_stream
    for fn, args in calls:
        check(fn(*args, stream))
    return {"kv": st["kv"], "out": st["out"]} if "kv" in st else st["out"]


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if kind == "quantize":                                    # and back: the values are what is returned
        n = case["rows"] * case["k"]
        return {"bytes": n * (size[case["type"]] + 2 + 4) + 8 * case["rows"], "flops": 4 * n}
    if kind == "linear":
        n, k, m = case["rows"], case["k"], case["m"]
        act = 1 if case["act"] == "i8" else size[case["act"]]
        return {"bytes": k * m + 4 * m + n * k * act + n * m * size[case["out"]] + 4 * m * case["bias"], "flops": 2 * n * k * m}
    if kind == "rope":
        n, axes = case["batch"] * case["seq"], len(_dims(case))
        return {"bytes": n * (2 * case["heads"] * case["d"] * size[case["type"]] + 4 * axes) + 4 * case["d"] * case["norm"],
                "flops": n * case["heads"] * (3 * sum(_dims(case)) + 4 * case["d"] * case["norm"])}
    if kind == "cross":
        b, nq, h, d = case["batch"], case["nq"], case["heads"], case["d"]
        # half of the states, over the lengths that prepare draws
        share = {"none": 1.0, "len": (1 + (b - 1) / 2) / b, "holes": 0.75}[case["mask"]]
        n = case["nkv"] * share
        return {"bytes": b * d * 2 * (2 * nq * h + 2 * n * case["kv_heads"]), "flops": 4 * b * nq * n * h * d}
    b, nq, c, hd = case["batch"], case["nq"], case["c"], case["heads"] * case["d"]
    n = case["frames"] * case["height"] * case["width"]
    share = (1 + (b - 1) / 2) / b
    return {"bytes": b * (nq * c * 4 + n * c * 2 + n * 2 * hd * 2 + nq * hd * 2 + 8 * c) + 3 * hd * (c + 4),
            "flops": 2 * b * (nq + 2 * n) * c * hd + 4 * b * nq * n * share * hd}


# ---------------------------------------------------------------- the same in 64 bits
def _rows_in_8_bits(x):
    """rows in 64 bits: the integers nearest to x in steps of the largest / 127, and the steps, which are float32 numbers"""
    step = (torch.clamp(x.abs().max(dim=-1, keepdim=True).values, min=TINY) / 127).float().double()
    return torch.round(x / step), step


def _matrix(planes, rows, k):
    q, d = _unpack(planes, rows, k)
    return q.double(), d.double()


def _product(x, w):
    return torch.mm(x[0], w[0].T.contiguous()) * x[1] * w[1].T


def _turned(x, pos, dims, pairs, shared):
    """x (b, s, h, d), pos (b, n, s): each pair as a complex number times exp(i angle)"""
    out, n, at = x.clone(), sum(dims), 0
    for a, k in enumerate(dims):
        for j in range(k // 2):
            i = at // 2 + j
            angle = pos[:, a] * 10000.0 ** (-2.0 * i / n if shared else -2.0 * j / k)
            one, two = (2 * i, 2 * i + 1) if pairs == "adjacent" else (i, n // 2 + i)
            z = torch.complex(x[..., one], x[..., two]) * torch.polar(torch.ones_like(angle), angle)[:, :, None]
            out[..., one], out[..., two] = z.real, z.imag
        at += k
    return out


def _attended(q, k, v, keep):
    """one head at a time; q (b, nq, h, d), k, v (b, nkv, g, d), keep (b, nkv) or None"""
    out = torch.zeros_like(q)
    for b in range(q.shape[0]):
        at = slice(None) if keep is None else keep[b].nonzero()[:, 0]
        for h in range(q.shape[2]):
            g = h * k.shape[2] // q.shape[2]
            kk, vv = k[b, at, g], v[b, at, g]
            if len(kk):
                p = torch.softmax(torch.mm(q[b, :, h], kk.T.contiguous()) / math.sqrt(q.shape[-1]), -1)
                out[b, :, h] = torch.mm(p, vv)
    return out


def exact(case, seed):
    st = {k: v for k, v in prepare(case, seed).items() if k not in ("out", "planes")}
    d = {k: v.double() for k, v in st.items() if torch.is_tensor(v) and k not in ("weights", "wq", "wkv")}
    kind = case["kind"]
    if kind == "quantize":
        q, step = _rows_in_8_bits(d["x"])
        return q * step
    if kind == "linear":
        n, k, m = case["rows"], case["k"], case["m"]
        y = _product(_matrix(st["x"], n, k) if case["act"] == "i8" else _rows_in_8_bits(d["x"]), _matrix(st["weights"], m, k))
        return y + d["bias"] if "bias" in d else y
    if kind == "rope":
        x = d["x"]
        if "w" in d:
            x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + EPS) * d["w"]
        return _turned(x, d["pos"], _dims(case), case["pairs"], case["shared"])
    keep = None
    if "len" in d:
        keep = torch.arange((st["k"] if kind == "cross" else st["states"]).shape[1], device=DEV)[None] < d["len"][:, None]
    elif "valid" in d:
        keep = d["valid"] > 0
    if kind == "cross":
        return _attended(d["q"], d["k"], d["v"], keep)
    c, h, hd = case["c"], case["heads"], case["d"]
    x = d["x"] - d["x"].mean(-1, keepdim=True)
    x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + EPS) * (1 + d["scale"]) + d["shift"]
    q = _product(_rows_in_8_bits(x.reshape(-1, c)), _matrix(st["wq"], h * hd, c)).reshape(st["q"].shape)
    kv = _product(_rows_in_8_bits(d["states"].reshape(-1, c)), _matrix(st["wkv"], 2 * h * hd, c)).reshape(st["kv"].shape)
    head = lambda y, w: y / torch.sqrt((y ** 2).mean(-1, keepdim=True) + EPS) * w  # noqa: E731
    q = _turned(head(q, d["qw"]), d["qpos"][None], _block_dims(hd), "adjacent", False)
    k = _turned(head(kv[:, :, 0], d["kw"]), d["kpos"][None], _block_dims(hd), "adjacent", False)
    return {"kv": torch.stack([k, kv[:, :, 1]], 2), "out": _attended(q, k, kv[:, :, 1], keep)}
