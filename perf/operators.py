"""Performance cases of the 4-bit block-scaled (MXFP4) operators and of the
fused block norm: quantization, products with 4-bit weights, and the norms,
gate and residual around a block.

With `own` the calls a user makes of libtsk.so, else the same operators in
elementary torch operations. MXFP4 holds 32 values along a row as 4-bit
E2M1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) and one E8M0
byte E: each value is the number times 2^(E - 127). The split planes hold
rows of K / 2 bytes (value 2 i in byte i's low nibble), then rows of K / 32
scale bytes. Sizes are the models': 194 / 646 latent tokens of a 9 s / 30 s
clip, batches of 2, hidden 1024, MLPs of 4096 and 2816, T5 2048 and 5120; and
generic ones.
"""
import ctypes
import math

import torch

own = False
DEV = "cuda"
EPS = 1e-5


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # the activations of a text stream on their way into a 4-bit product: launch latency
        {"name": "quantize_text", "kind": "quantize", "type": "f32", "rows": 77, "k": 1024},
        # the hidden state of the SwiGLU MLP at 30 s, kept in bf16
        {"name": "quantize_mlp_30s", "kind": "quantize", "type": "bf16", "rows": 1292, "k": 2816},
        # a large weight matrix, once at load
        {"name": "quantize_weights", "kind": "quantize", "type": "f32", "rows": 8192, "k": 8192},
        # adaLN of one conditioning row: a single token against 4-bit weights
        {"name": "linear_one_row", "kind": "linear", "act": "bf16", "rows": 1, "k": 1024, "m": 6144, "out": "f32", "bias": True},
        # a few rows against a large layer: the weights' bytes
        {"name": "linear_few_rows", "kind": "linear", "act": "bf16", "rows": 8, "k": 8192, "m": 8192, "out": "bf16", "bias": False},
        # the MLP's first projection at 9 s on f32 activations, weights alone in 4 bits
        {"name": "linear_9s", "kind": "linear", "act": "f32", "rows": 388, "k": 1024, "m": 4096, "out": "f32", "bias": True},
        # T5's projection back to its width over several texts, ragged in rows and outputs
        {"name": "linear_ragged", "kind": "linear", "act": "bf16", "rows": 2047, "k": 5120, "m": 2050, "out": "bf16", "bias": True},
        # the MLP's second projection at 30 s, both operands in 4 bits: long rows, few tiles
        {"name": "linear_4bit_30s", "kind": "linear", "act": "mxfp4", "rows": 1292, "k": 4096, "m": 1024, "out": "f32", "bias": True},
        # a large product of two 4-bit operands: the matrix unit's rate
        {"name": "linear_4bit_large", "kind": "linear", "act": "mxfp4", "rows": 8192, "k": 8192, "m": 8192, "out": "bf16", "bias": False},
        # gate and residual of the attention, LayerNorm and modulation before the MLP, one block at 9 s
        {"name": "norm_9s", "kind": "norm", "norm": "layer", "post": False, "type": "f32", "batch": 2, "seq": 194, "c": 1024,
         "mod": "batch"},
        # a block with RMS norms on both sides of its branch over many bf16 rows: memory
        {"name": "norm_sandwich", "kind": "norm", "norm": "rms", "post": True, "type": "bf16", "batch": 4, "seq": 4096, "c": 4096,
         "mod": "none"},
        # residual, norm and modulation straight into the 4-bit operand of the MLP's first projection at 30 s
        {"name": "norm_linear_30s", "kind": "norm_linear", "norm": "layer", "post": False, "type": "f32", "batch": 2, "seq": 646,
         "c": 1024, "mod": "token", "m": 4096},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "linear", "norm", "norm", "norm_linear"])
    if kind == "quantize":
        k = 32 * _log(rng, 1, 256)
        return {"kind": kind, "type": rng.choice(["f32", "bf16"]), "rows": _log(rng, 1, 8192), "k": k}
    if kind == "linear":
        act = rng.choice(["bf16", "f32", "mxfp4", "mxfp4"])
        k, m = 32 * _log(rng, 2, 256), _log(rng, 16, 8192)
        # both sides of a product of 16-bit activations cost more than of 4-bit ones
        most = max(1, min(8192, (8192 if act == "mxfp4" else 1024) * 8192 * 8192 // (k * m)))
        return {"kind": kind, "act": act, "rows": _log(rng, 1, most), "k": k, "m": m, "out": rng.choice(["f32", "bf16"]),
                "bias": rng.random() < 0.5}
    case = {"kind": kind, "norm": rng.choice(["layer", "rms"]), "post": rng.random() < 0.5, "type": rng.choice(["f32", "bf16"]),
            "batch": rng.choice([1, 2, 4]), "seq": _log(rng, 1, 4096), "mod": rng.choice(["none", "batch", "token"])}
    case["c"] = _log(rng, 16, 4096) if kind == "norm" else 32 * _log(rng, 2, 64)
    case["seq"] = max(1, min(case["seq"], 4096 * 4096 // (case["batch"] * case["c"])))
    return case if kind == "norm" else case | {"m": _log(rng, 16, 4096)}


# ---------------------------------------------------------------- MXFP4 in elementary operations
_NUMBERS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _codes(x):
    """f32 rows (R, K): 4-bit codes (R, K / 32, 32) and scale bytes (R, K / 32), int32"""
    b = x.reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1)                                    # NaN where the block holds one
    # the exponent byte of amax, two less; 2^-127 at least (zeros and the smallest numbers)
    byte = ((top.view(torch.int32) >> 23) - 2).clamp(min=0)
    back = ((254 - byte) << 23).view(torch.float32)           # 2^(127 - byte)
    a = b.abs() * back[..., None]
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5.0).int())
    bad = ~torch.isfinite(top)
    code = torch.where(bad[..., None], 0, code + 8 * torch.signbit(b).int())
    return code, torch.where(bad, 255, byte)


def _values(code, byte):
    """the f32 numbers that codes (R, B, 32) and scale bytes (R, B) stand for"""
    numbers = torch.tensor(_NUMBERS + [-v for v in _NUMBERS], device=code.device)
    bits = torch.where(byte == 0, 0x00400000, byte << 23)     # 2^-127 is below the normal numbers
    scale = torch.where(byte == 255, math.nan, bits.int().view(torch.float32))
    return (numbers[code.long()] * scale[..., None]).reshape(code.shape[0], -1)


def _pack(code, byte):
    """the split planes, one array of bytes"""
    c = code.reshape(code.shape[0], -1)
    return torch.cat([(c[:, 0::2] | (c[:, 1::2] << 4)).to(torch.uint8).reshape(-1), byte.to(torch.uint8).reshape(-1)])


def _unpack(planes, rows, k):
    q = planes[:rows * k // 2].reshape(rows, k // 2).int()
    return torch.stack([q & 15, q >> 4], -1).reshape(rows, k // 32, 32), planes[rows * k // 2:].reshape(rows, k // 32).int()


# ---------------------------------------------------------------- inputs
class _Rand:
    """seeded inputs, made on the GPU"""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(1 + int(seed))

    def __call__(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.g, device=DEV, dtype=torch.float32) * std


def _typed(x, typ):
    return x.bfloat16() if typ == "bf16" else x


def _padded(rows, m, typ):
    """an output of `rows` rows whose strides are multiples of 16 bytes, as a view of m columns"""
    return torch.empty(rows, (m + 7) // 8 * 8, dtype=torch.bfloat16 if typ == "bf16" else torch.float32, device=DEV)[:, :m]


def _mxfp4(x):
    return _pack(*_codes(x))


def _norm_inputs(case, r):
    b, s, c = case["batch"], case["seq"], case["c"]
    n = {"batch": 1, "token": s}.get(case["mod"])
    st = {"x": _typed(r(b, s, c, std=2.0) + 0.3, case["type"]), "y": _typed(r(b, s, c), case["type"]), "gate": None, "scale": None,
          "shift": None, "post_w": 1 + r(c, std=0.1) if case["post"] else None, "w": None}
    if n:
        st.update(gate=r(b, n, c, std=0.5), scale=r(b, n, c, std=0.3), shift=r(b, n, c, std=0.3))
    else:
        st["w"] = 1 + r(c, std=0.1)
    return st


def prepare(case, seed):
    r, kind, st = _Rand(seed), case["kind"], {"case": case}
    if kind == "quantize":
        n, k = case["rows"], case["k"]
        # rows of different sizes, as activations and weight rows have
        st["x"] = _typed(r(n, k) * torch.exp(r(n, 1)), case["type"])
        st["planes"] = torch.empty(n * k // 2 + n * k // 32, dtype=torch.uint8, device=DEV)
        st["out"] = torch.empty(n, k, device=DEV)
        return st
    if kind == "linear":
        n, k, m = case["rows"], case["k"], case["m"]
        x = r(n, k)
        st["x"] = _mxfp4(x) if case["act"] == "mxfp4" else _typed(x, case["act"])
        st["bias"] = r(m, std=0.02) if case["bias"] else None
        st["weights"] = _mxfp4(r(m, k, std=k ** -0.5))
        st["out"] = _padded(n, m, case["out"])
        return st
    st.update(_norm_inputs(case, r))
    st["res"] = torch.empty_like(st["x"])
    if kind == "norm":
        st["h"] = torch.empty_like(st["x"])
        return st
    n, c, m = case["batch"] * case["seq"], case["c"], case["m"]
    st["weights"] = _mxfp4(r(m, c, std=c ** -0.5))
    st["planes"] = torch.empty(n * c // 2 + n * c // 32, dtype=torch.uint8, device=DEV)
    st["out"] = _padded(n, m, "bf16")
    return st


# ---------------------------------------------------------------- one pass
def _plain_norm(x, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _plain_block(st):
    case = st["case"]
    y = st["y"].float()
    if case["post"]:
        y = _plain_norm(y, case["norm"]) * st["post_w"]
    res = st["x"].float() + (y if st["gate"] is None else st["gate"] * y)
    res = _typed(res, case["type"])
    h = _plain_norm(res.float(), case["norm"])
    if st["w"] is not None:
        h = h * st["w"]
    if st["scale"] is not None:
        h = h * (1 + st["scale"]) + st["shift"]
    return res, h


def _plain(st):
    case = st["case"]
    if case["kind"] == "quantize":
        return _values(*_codes(st["x"].float()))
    if case["kind"] == "linear":
        n, k, m = case["rows"], case["k"], case["m"]
        # f32 activations are multiplied as bf16, like those of bf16 weights
        x = _values(*_unpack(st["x"], n, k)) if case["act"] == "mxfp4" else st["x"].bfloat16().float()
        y = x @ _values(*_unpack(st["weights"], m, k)).T
        return _typed(y if st["bias"] is None else y + st["bias"], case["out"])
    res, h = _plain_block(st)
    if case["kind"] == "norm":
        return {"res": res, "h": _typed(h, case["type"])}
    c, m = case["c"], case["m"]
    h = _values(*_codes(h.reshape(-1, c)))
    return {"res": res, "out": (h @ _values(*_unpack(st["weights"], m, c)).T).bfloat16()}


def _plan(st):
    """the descriptors of the calls, built once for the buffers that the program keeps"""
    from __graft_entry__ import load_tsk
    t = load_tsk()
    t.init(0)
    types = {torch.float32: t.F32, torch.bfloat16: t.BF16}
    lib, case = t.load(), st["case"]

    def d(x):
        return None if x is None else ctypes.pointer(t.desc(x, types[x.dtype]))

    def planes(x, rows, k):
        return ctypes.pointer(t.desc(t.SplitMXFP4(x, k, rows), t.MXFP4_SPLIT))

    if case["kind"] == "quantize":
        q = planes(st["planes"], case["rows"], case["k"])
        return t.check, [(lib.tsk_mxfp4_quantize, (d(st["x"]), q)), (lib.tsk_mxfp4_dequantize, (q, d(st["out"])))]
    if case["kind"] == "linear":
        n, k, m = case["rows"], case["k"], case["m"]
        x = planes(st["x"], n, k) if case["act"] == "mxfp4" else d(st["x"])
        return t.check, [(lib.tsk_mul_mat, (planes(st["weights"], m, k), x, d(st["bias"]), d(st["out"])))]
    kind = t.NORM_LAYER if case["norm"] == "layer" else t.NORM_RMS
    p = t.BlockNormParams()
    p.post_norm, p.post_eps, p.post_w = kind if case["post"] else t.NORM_NONE, EPS, d(st["post_w"])
    p.gate, p.res_scale = d(st["gate"]), 1.0
    p.pre_norm, p.pre_eps, p.pre_w, p.scale, p.shift = kind, EPS, d(st["w"]), d(st["scale"]), d(st["shift"])
    if case["kind"] == "norm":
        return t.check, [(lib.tsk_block_norm, (d(st["x"]), d(st["y"]), ctypes.pointer(p), d(st["res"]), d(st["h"])))]
    n, c, m = case["batch"] * case["seq"], case["c"], case["m"]
    b, s = case["batch"], case["seq"]
    h = planes(st["planes"], n, c)                            # [c, s, b] for the norm, [c, n] for the product: the same rows
    h3 = planes(st["planes"], n, c)
    h3.contents.ne[1], h3.contents.ne[2] = s, b
    return t.check, [(lib.tsk_block_norm, (d(st["x"]), d(st["y"]), ctypes.pointer(p), d(st["res"]), h3)),
                     (lib.tsk_mul_mat, (planes(st["weights"], m, c), h, None, d(st["out"])))]


def _own(st):
    if "plan" not in st:
        st["plan"] = _plan(st)
    check, calls = st["plan"]
    stream = torch.cuda.current_stream().cuda_stream
    for fn, args in calls:
        check(fn(*args, stream))
    if "h" in st:
        return {"res": st["res"], "h": st["h"]}
    return {"res": st["res"], "out": st["out"]} if "res" in st else st["out"]


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    per = 2 if case.get("type") == "bf16" else 4
    if kind == "quantize":                                    # and back: the values are what is returned
        n = case["rows"] * case["k"]
        return {"bytes": n * (per + 2 * 17 / 32 + 4), "flops": 4 * n}
    if kind == "linear":
        n, k, m = case["rows"], case["k"], case["m"]
        act = {"bf16": 2, "f32": 4, "mxfp4": 17 / 32}[case["act"]]
        return {"bytes": k * m * 17 / 32 + n * k * act + n * m * (2 if case["out"] == "bf16" else 4) + 4 * m * case["bias"],
                "flops": 2 * n * k * m}
    rows, c = case["batch"] * case["seq"], case["c"]
    mod = 3 * 4 * c * {"none": 0, "batch": case["batch"], "token": rows}[case["mod"]]
    if kind == "norm":
        return {"bytes": 4 * rows * c * per + mod, "flops": 16 * rows * c}
    m = case["m"]
    return {"bytes": 3 * rows * c * per + mod + 17 / 32 * c * (2 * rows + m) + 2 * rows * m, "flops": 2 * rows * c * m + 16 * rows * c}


# ---------------------------------------------------------------- the same in 64 bits
def _number(c):
    """E2M1 codes: sign, two exponent bits (bias 1), one mantissa bit"""
    e, f = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e == 0, 0.5 * f, (1 + 0.5 * f) * torch.exp2(e.double() - 1))
    return torch.where(c >= 8, -v, v)


def _matrix(planes, rows, k):
    q = planes[:rows * (k // 2)].long().reshape(rows, k // 2)
    v = torch.empty(rows, k, dtype=torch.float64, device=DEV)
    v[:, 0::2], v[:, 1::2] = _number(q % 16), _number(q // 16)
    s = planes[rows * (k // 2):].double().reshape(rows, k // 32)
    return v * torch.exp2(s - 127).repeat_interleave(32, dim=1)


def _rounded(x):
    """rows in 64 bits to the nearest MXFP4 values: steps of 0.5 below 2, 1 below 4, 2 above, at most 6"""
    b = x.reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
    e = e + (torch.exp2(e + 1) <= top).double() - (torch.exp2(e) > top).double()      # log2 next to a power of two
    s = torch.exp2(torch.where(top > 0, e - 2, -127.0).clamp(min=-127.0))
    a = b.abs() / s
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.sign(b) * (torch.round(a / step) * step).clamp(max=6.0) * s).reshape(x.shape)


def _normed(x, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)


def exact(case, seed):
    st = {k: v for k, v in prepare(case, seed).items() if k not in ("out", "res", "h", "planes")}
    d = {k: v.double() for k, v in st.items() if torch.is_tensor(v)}
    if case["kind"] == "quantize":
        return _rounded(d["x"])
    if case["kind"] == "linear":
        n, k, m = case["rows"], case["k"], case["m"]
        x = _matrix(st["x"], n, k) if case["act"] == "mxfp4" else st["x"].to(torch.bfloat16).double()
        y = torch.mm(x, _matrix(st["weights"], m, k).T.contiguous())
        return y + d["bias"] if "bias" in d else y
    y = _normed(d["y"], case["norm"]) * d["post_w"] if case["post"] else d["y"]
    res = d["x"] + (d["gate"] * y if "gate" in d else y)
    kept = res.to(torch.bfloat16).double() if case["type"] == "bf16" else res
    h = _normed(kept, case["norm"])
    h = h * d["w"] if "w" in d else h * (1 + d["scale"]) + d["shift"]
    if case["kind"] == "norm":
        return {"res": res, "h": h}
    c, m = case["c"], case["m"]
    return {"res": res, "out": torch.mm(_rounded(h.reshape(-1, c)), _matrix(st["weights"], m, c).T.contiguous())}
