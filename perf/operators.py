"""The 8-bit block operators' cases: row norms that write 8-bit rows with scales, row quantisation, and
matrix products (16-bit and 8-bit operands) whose epilogue adds a bias, applies an activation or a gate
and adds a residual.

``run`` has each operator twice: in elementary torch operations in 32 bits (``own`` false), and as the
calls a user makes of ``glypr_b200.api`` (``own`` true).  The definitions, with q(v) a row's 8-bit form
(scale = max(max|v| / top, 2^-100), codes = round(v / scale), top = 448 for e4m3 and 127 for int8):

  norm      h = (residual + x~) * layer_scalar, x~ = x rms(x) post_gain or x;  q(h rms(h) gain);
            rms(v) = 1 / sqrt(mean(v^2) + eps)
  quantize  q(x)
  linear    y = act(x w^T s + bias) [* (x w_up^T s_up + bias_up)] + residual; 8-bit operands have a scale
            per row of x and of w, 16-bit ones none
  block     an int8 feed-forward half of a layer: norm -> gated linear -> quantize -> linear

Codes of 8 bits come back as e4m3 tensors beside their scales; int8 codes stay inside a block.
"""
import math

import torch

own = False

EPS = 1e-6
FLOOR = 2.0 ** -100
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn,
         "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "i8": 1}
TOP = {"e4m3": 448.0, "i8": 127.0}


# ------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one token through a norm: nothing but latency
        {"name": "norm_one_row", "op": "norm", "m": 1, "h": 768, "x": "f16", "res": "bf16", "post": True},
        # a launch chunk of 262,144 tokens at the model's width: the sandwich norm between two sublayers
        {"name": "norm_chunk", "op": "norm", "m": 262144, "h": 768, "x": "f16", "res": "bf16", "post": True},
        # an odd width (no row but the first is aligned), an odd row count, plain pre-norm with its addition
        {"name": "norm_odd", "op": "norm", "m": 10007, "h": 1543, "x": "bf16", "res": "bf16", "post": False},
        # one 512-token sequence's feed-forward activations on their way to the down projection
        {"name": "quantize_sequence", "op": "quantize", "m": 512, "h": 1152, "x": "f16"},
        # the same for a half launch chunk
        {"name": "quantize_chunk", "op": "quantize", "m": 131072, "h": 1152, "x": "f16"},
        # one token, gate and up projections of the model's width: latency again
        {"name": "linear_one_token", "op": "linear", "dtype": "bf16", "m": 1, "n": 1152, "k": 768, "out": "bf16",
         "act": "gelu_tanh", "gated": True, "bias": False, "res": False},
        # one 512-token sequence, a biased projection added to the residual stream
        {"name": "linear_sequence", "op": "linear", "dtype": "f16", "m": 512, "n": 768, "k": 768, "out": "f16",
         "act": "none", "gated": False, "bias": True, "res": True},
        # a half launch chunk, the down projection onto the residual stream
        {"name": "linear_chunk", "op": "linear", "dtype": "bf16", "m": 131072, "n": 768, "k": 1152, "out": "bf16",
         "act": "none", "gated": False, "bias": True, "res": True},
        # a few rows against a large 8-bit weight of an odd number of rows: the weight's bytes
        {"name": "linear8_few_rows", "op": "linear", "dtype": "e4m3", "m": 3, "n": 8191, "k": 4096, "out": "bf16",
         "act": "silu", "gated": False, "bias": True, "res": False},
        # the gate and up projections of a half launch chunk in int8
        {"name": "linear8_gated_chunk", "op": "linear", "dtype": "i8", "m": 131072, "n": 1152, "k": 768, "out": "f16",
         "act": "gelu_tanh", "gated": True, "bias": False, "res": False},
        # a wide layer: the tensor cores' rate
        {"name": "linear8_wide", "op": "linear", "dtype": "e4m3", "m": 16384, "n": 4096, "k": 4096, "out": "bf16",
         "act": "gelu_erf", "gated": False, "bias": True, "res": True},
        # the operators together, as a layer's feed-forward half runs them on 64 sequences of 512 tokens
        {"name": "block_int8", "op": "block", "m": 32768, "h": 768, "f": 1152},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "linear", "linear", "linear", "block"])
    m = _log(rng, 1, 131072)
    if op in ("norm", "quantize"):
        h = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            h = max(64, h // 8 * 8)
        m = max(1, min(m, 262144 * 768 // h))
        x = rng.choice(["f16", "bf16", "f32"])
        if op == "quantize":
            return {"op": op, "m": m, "h": h, "x": x}
        return {"op": op, "m": m, "h": h, "x": x, "res": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "post": rng.random() < 0.5}
    if op == "block":
        h, f = _log(rng, 256, 2048) // 16 * 16, _log(rng, 256, 4096) // 16 * 16
        return {"op": op, "m": max(1, min(m, 32768 * 768 * 4608 // (h * f))), "h": h, "f": f}
    dtype = rng.choice(["f16", "bf16", "e4m3", "i8"])
    gated = rng.random() < 0.3
    n, k = _log(rng, 64, 8192), _log(rng, 64, 8192)
    if rng.random() < 0.6:
        n, k = max(64, n // 16 * 16), max(64, k // 16 * 16)
    m = max(1, min(m, 16384 * 4096 * 4096 // (n * k * (2 if gated else 1)), 402653184 // max(n, k)))
    return {"op": op, "dtype": dtype, "m": m, "n": n, "k": k, "out": rng.choice(["bf16", "f16", "f32"]),
            "act": rng.choice(["none", "relu", "silu", "gelu_tanh", "gelu_erf"]) if not gated
            else rng.choice(["silu", "gelu_tanh", "gelu_erf"]),
            "gated": gated, "bias": rng.random() < 0.5, "res": rng.random() < 0.5}


def work(case):
    """Each input once, each output once; two operations per product term."""
    m, op = case["m"], case["op"]
    if op == "norm":
        h = case["h"]
        # x, residual in, h out, codes, gains, scales; ~ 12 operations an element
        per = SIZE[case["x"]] + 2 * SIZE[case["res"]] + 1
        return {"bytes": m * h * per + 4 * h * (2 if case["post"] else 1) + 4 * m, "flops": 12.0 * m * h}
    if op == "quantize":
        return {"bytes": m * case["h"] * (SIZE[case["x"]] + 1) + 4 * m, "flops": 4.0 * m * case["h"]}
    if op == "linear":
        n, k, e, o = case["n"], case["k"], SIZE[case["dtype"]], SIZE[case["out"]]
        two = 2 if case["gated"] else 1
        b = m * k * e + two * n * k * e + m * n * o * (2 if case["res"] else 1) + (two * 4 * n if case["bias"] else 0)
        b += (4 * m + two * 4 * n) if e == 1 else 0
        return {"bytes": b, "flops": 2.0 * m * n * k * two}
    h, f = case["h"], case["f"]
    # x, residual in; h and the half's output out; three weights: what goes between them is the path's own
    return {"bytes": m * h * (2 + 2 + 2 + 2) + 3 * h * f + 4 * (2 * h + 2 * f + h), "flops": 6.0 * m * h * f}


# ------------------------------------------------------------------------------------- inputs

def _pitch(cols, size):
    """Row pitch in elements: rows of matrix-product operands start on 16-byte boundaries."""
    a = 16 // size
    return (cols + a - 1) // a * a


def _rows(g, m, k, spread=0.5):
    """Rows of normal values whose sizes differ as tokens' do, a few columns larger than the rest."""
    v = torch.randn((m, k), generator=g, device="cuda")
    v *= torch.exp(spread * torch.randn((m, 1), generator=g, device="cuda"))
    v[:, :: 97] *= 4.0
    return v


def _padded(v, dtype):
    m, k = v.shape
    buf = torch.zeros((m, _pitch(k, SIZE[dtype])), dtype=TYPES[dtype], device="cuda")
    buf[:, :k] = v.to(TYPES[dtype])
    return buf[:, :k]


def _codes8(v, dtype):
    """8-bit rows and scales of an operand, made as a user's program holds them (weights laid out once)."""
    s = (v.abs().amax(1) / TOP[dtype]).clamp_min(FLOOR)
    c = v / s[:, None]
    return _padded(c.round() if dtype == "i8" else c, dtype), s


def _operand(g, m, k, dtype, scale):
    v = _rows(g, m, k) * scale
    if SIZE[dtype] == 2:
        return _padded(v, dtype), None
    return _codes8(v, dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, m = case["op"], case["m"]
    s = {"case": case}

    def empty(rows, cols, dtype):
        return torch.empty((rows, cols), dtype=TYPES[dtype], device="cuda")

    def gain(n):
        return 1.0 + 0.2 * torch.randn(n, generator=g, device="cuda")

    if op == "norm":
        h = case["h"]
        s.update(x=_rows(g, m, h).to(TYPES[case["x"]]), res=(2 * _rows(g, m, h)).to(TYPES[case["res"]]), gain=gain(h),
                 post=gain(h) if case["post"] else None, h=empty(m, h, case["res"]), q=empty(m, h, "e4m3"),
                 scale=torch.empty(m, device="cuda"))
    elif op == "quantize":
        s.update(x=_rows(g, m, case["h"]).to(TYPES[case["x"]]), q=empty(m, case["h"], "e4m3"),
                 scale=torch.empty(m, device="cuda"))
    elif op == "linear":
        n, k, d = case["n"], case["k"], case["dtype"]
        s["x"], s["xs"] = _operand(g, m, k, d, 0.5)
        s["w"], s["ws"] = _operand(g, n, k, d, 1.5 / math.sqrt(k))
        s["wu"], s["wus"] = _operand(g, n, k, d, 1.5 / math.sqrt(k)) if case["gated"] else (None, None)
        s["b"] = 0.3 * torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        s["bu"] = 0.3 * torch.randn(n, generator=g, device="cuda") if case["bias"] and case["gated"] else None
        s["res"] = torch.randn((m, n), generator=g, device="cuda").to(TYPES[case["out"]]) if case["res"] else None
        s["y"] = empty(m, n, case["out"])
    else:
        h, f = case["h"], case["f"]
        s.update(x=_rows(g, m, h).to(torch.float16), res=(2 * _rows(g, m, h)).to(torch.bfloat16), gain=gain(h),
                 post=gain(h))
        for name, n, k in (("wg", f, h), ("wu", f, h), ("wd", h, f)):
            s[name], s[name + "s"] = _operand(g, n, k, "i8", 1.5 / math.sqrt(k))
        s.update(h=empty(m, h, "bf16"), q=empty(m, h, "i8"), scale=torch.empty(m, device="cuda"), a=empty(m, f, "f16"),
                 qa=empty(m, f, "i8"), sa=torch.empty(m, device="cuda"), y=empty(m, h, "f16"))
    return s


# ------------------------------------------------------------------------------------- plain form

def _rms(v):
    return 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)


def _quantized(v, dtype):
    s = (v.abs().amax(1) / TOP[dtype]).clamp_min(FLOOR)
    c = v / s[:, None]
    return (c.round() if dtype == "i8" else c.to(TYPES[dtype])), s


def _act(v, kind):
    if kind == "relu":
        return v.clamp_min(0)
    if kind == "silu":
        return v / (1 + torch.exp(-v))
    if kind == "gelu_tanh":
        return v / (1 + torch.exp(-2 * 0.7978845608028654 * (v + 0.044715 * v * v * v)))
    if kind == "gelu_erf":
        return 0.5 * v * torch.erfc(-0.7071067811865476 * v)
    return v


def _norm_plain(s, scalar=1.0):
    x = s["x"].float()
    if s["post"] is not None:
        x = x * _rms(x) * s["post"]
    h = (s["res"].float() + x) * scalar
    return h, h * _rms(h) * s["gain"]


def _product(x, xs, w, ws, b):
    v = x.float() @ w.float().T
    if xs is not None:
        v = v * xs[:, None] * ws
    return v if b is None else v + b


def _plain(s):
    c = s["case"]
    if c["op"] == "norm":
        h, n = _norm_plain(s)
        q, scale = _quantized(n, "e4m3")
        return {"h": h.to(s["res"].dtype), "q": q, "scale": scale}
    if c["op"] == "quantize":
        q, scale = _quantized(s["x"].float(), "e4m3")
        return {"q": q, "scale": scale}
    if c["op"] == "linear":
        y = _act(_product(s["x"], s["xs"], s["w"], s["ws"], s["b"]), c["act"])
        if c["gated"]:
            y = y * _product(s["x"], s["xs"], s["wu"], s["wus"], s["bu"])
        if s["res"] is not None:
            y = y + s["res"].float()
        return {"y": y.to(TYPES[c["out"]])}
    h, n = _norm_plain(s)
    q, scale = _quantized(n, "i8")
    a = _act(_product(q, scale, s["wg"], s["wgs"], None), "gelu_tanh") * _product(q, scale, s["wu"], s["wus"], None)
    qa, sa = _quantized(a, "i8")
    return {"h": h.to(torch.bfloat16), "y": _product(qa, sa, s["wd"], s["wds"], None).to(torch.float16)}


# ------------------------------------------------------------------------------------- the framework's

def _p(t):
    return 0 if t is None else t.data_ptr()


def _own(s):
    from glypr_b200 import api
    c = s["case"]
    st = torch.cuda.current_stream().cuda_stream
    dt = api.DTYPES
    if c["op"] == "norm":
        api.norm_residual_q8(c["m"], c["h"], s["x"].data_ptr(), dt[c["x"]], s["q"].data_ptr(), dt["e4m3"],
                             s["scale"].data_ptr(), gain=s["gain"].data_ptr(), post_gain=_p(s["post"]),
                             residual=s["res"].data_ptr(), h=s["h"].data_ptr(), h_dtype=dt[c["res"]], eps=EPS, stream=st)
        return {"h": s["h"], "q": s["q"], "scale": s["scale"]}
    if c["op"] == "quantize":
        api.quantize_rows(c["m"], c["h"], s["x"].data_ptr(), dt[c["x"]], s["q"].data_ptr(), dt["e4m3"],
                          s["scale"].data_ptr(), stream=st)
        return {"q": s["q"], "scale": s["scale"]}
    if c["op"] == "linear":
        api.linear(c["m"], c["n"], c["k"], dt[c["dtype"]], s["x"].data_ptr(), s["w"].data_ptr(), s["y"].data_ptr(),
                   dt[c["out"]], ldx=s["x"].stride(0), ldw=s["w"].stride(0), x_scale=_p(s["xs"]), w_scale=_p(s["ws"]),
                   w_up=_p(s["wu"]), w_up_scale=_p(s["wus"]), bias=_p(s["b"]), bias_up=_p(s["bu"]),
                   activation=api.ACTIVATIONS[c["act"]], residual=_p(s["res"]), stream=st)
        return {"y": s["y"]}
    m, h, f = c["m"], c["h"], c["f"]
    api.norm_residual_q8(m, h, s["x"].data_ptr(), dt["f16"], s["q"].data_ptr(), dt["i8"], s["scale"].data_ptr(),
                         gain=s["gain"].data_ptr(), post_gain=s["post"].data_ptr(), residual=s["res"].data_ptr(),
                         h=s["h"].data_ptr(), h_dtype=dt["bf16"], eps=EPS, stream=st)
    api.linear(m, f, h, dt["i8"], s["q"].data_ptr(), s["wg"].data_ptr(), s["a"].data_ptr(), dt["f16"],
               x_scale=s["scale"].data_ptr(), w_scale=s["wgs"].data_ptr(), w_up=s["wu"].data_ptr(),
               w_up_scale=s["wus"].data_ptr(), activation=api.ACTIVATIONS["gelu_tanh"], stream=st)
    api.quantize_rows(m, f, s["a"].data_ptr(), dt["f16"], s["qa"].data_ptr(), dt["i8"], s["sa"].data_ptr(), stream=st)
    api.linear(m, h, f, dt["i8"], s["qa"].data_ptr(), s["wd"].data_ptr(), s["y"].data_ptr(), dt["f16"],
               x_scale=s["sa"].data_ptr(), w_scale=s["wds"].data_ptr(), stream=st)
    return {"h": s["h"], "y": s["y"]}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------- 64 bits

def _round_e4m3(v):
    """Nearest e4m3 value (3 fraction bits, exponents from -6, largest 448), ties to even."""
    _, e = torch.frexp(v)  # |v| in [2^(e-1), 2^e)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp_min(-6) - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _quantized64(v, dtype):
    s = torch.clamp(torch.amax(torch.abs(v), dim=1) / TOP[dtype], min=FLOOR)
    c = v / s.unsqueeze(1)
    return (torch.round(c) if dtype == "i8" else _round_e4m3(c)), s


def _act64(v, kind):
    if kind == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if kind == "silu":
        return v * torch.special.expit(v)
    if kind == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if kind == "gelu_erf":
        return v * torch.special.ndtr(v)
    return v


def _norm64(x, post, res, gain):
    def rms(v):
        return v * torch.rsqrt(torch.sum(v * v, dim=1, keepdim=True) / v.shape[1] + EPS)
    h = res + (rms(x) * post if post is not None else x)
    return h, rms(h) * gain


def _linear64(x, xs, w, ws, b):
    v = torch.matmul(x.double(), w.double().t())
    if xs is not None:
        v = xs.double().unsqueeze(1) * v * ws.double().unsqueeze(0)
    return v if b is None else v + b.double()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]

    def wide(t):
        return None if t is None else t.double()

    if op == "norm":
        h, n = _norm64(wide(s["x"]), wide(s["post"]), wide(s["res"]), wide(s["gain"]))
        q, scale = _quantized64(n, "e4m3")
        return {"h": h, "q": q, "scale": scale}
    if op == "quantize":
        q, scale = _quantized64(wide(s["x"]), "e4m3")
        return {"q": q, "scale": scale}
    if op == "linear":
        y = _act64(_linear64(s["x"], s["xs"], s["w"], s["ws"], s["b"]), case["act"])
        if case["gated"]:
            y = y * _linear64(s["x"], s["xs"], s["wu"], s["wus"], s["bu"])
        return {"y": y + wide(s["res"]) if s["res"] is not None else y}
    h, n = _norm64(wide(s["x"]), wide(s["post"]), wide(s["res"]), wide(s["gain"]))
    q, scale = _quantized64(n, "i8")
    a = _act64(_linear64(q, scale, s["wg"], s["wgs"], None), "gelu_tanh") * _linear64(q, scale, s["wu"], s["wus"], None)
    qa, sa = _quantized64(a, "i8")
    return {"h": h, "y": _linear64(qa, sa, s["wd"], s["wds"], None)}
