"""The 8-bit row operators and the matrix product with a full epilogue (glp_norm_residual_q8,
glp_quantize_rows, glp_linear) against plain 64-bit implementations, at the sizes, pitches,
alignments and values where they can go wrong.

Tolerances, from the arithmetic (u = half an ulp of the output type: f16 2^-11, bf16 2^-8, f32 2^-24):

* h: one rounding of a value computed in f32 from rows of at most 32,768 elements summed in
  partial sums: u |h| + 2^-18 (|residual| + |x~|), plus half an f16 subnormal step.
* scale: 2^-18 relative (the row's sum and one division).
* codes: half a step of the row's own grid, plus 2^-10 of a step for values that lie within the
  f32 error of a rounding boundary, plus 2^-17 for the value itself, relative to |residual| + |x~|
  carried through the norm (a sum that cancels keeps its terms' errors): int8 steps are `scale`, e4m3
  steps 2^-3 of a binade, at least 2^-9 * scale.
* linear: the K products and their sum, in f32 in any order, each addition off by at most 2^-23 of
  the sum of magnitudes: (K + 8) 2^-23 sum |x||w|; int8 sums are exact.  Activations have slopes of
  at most 1.2 and a relative error of at most 2^-15 (an exponential of arguments up to 88, whose own
  error and its argument's rounding are each |argument| 2^-23, and a quotient);
  a gated product adds both factors' errors.  Then u |y| and half an f16 subnormal step.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from glypr_b200 import api

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = api.DTYPES
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8,
         "e4m3": torch.float8_e4m3fn}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}
TOP = {"i8": 127.0, "e4m3": 448.0}
FLOOR = 2.0 ** -100
EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def _lib():
    api.load_library()
    yield
    assert api.kernel_status(0) == 0


def buffer(rows, cols, dtype, pad=0, offset=0, fill=None):
    """A [rows, cols] view with `pad` extra elements per row and a base `offset` elements in."""
    ld = cols + pad
    flat = torch.zeros(offset + rows * ld + 32, dtype=torch.uint8 if dtype in ("i8", "e4m3") else TORCH[dtype],
                       device="cuda")
    if fill is not None:
        flat.fill_(fill)
    v = flat[offset:offset + rows * ld].view(rows, ld)[:, :cols]
    return v.view(TORCH[dtype]) if dtype in ("i8", "e4m3") else v


def filled(values, dtype, pad=0, offset=0):
    v = buffer(values.shape[0], values.shape[1], dtype, pad, offset)
    v.copy_(values.to(TORCH[dtype]))
    return v


def ptr(t):
    return 0 if t is None else t.data_ptr()


def rows_of(m, h, seed, spread=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    v = torch.randn((m, h), generator=g, device="cuda")
    return v * torch.exp(spread * torch.randn((m, 1), generator=g, device="cuda"))


def check_codes(q, scale, want, dtype, mag=None):
    """codes * scale against the 64-bit rows they stand for; mag: the magnitudes of the terms that
    `want` is a sum of."""
    want = want.double()
    mag = want.abs() if mag is None else mag
    s_want = (want.abs().amax(1) / TOP[dtype]).clamp_min(FLOOR)
    s = scale.double()
    assert ((s - s_want).abs() <= 2.0 ** -18 * s_want).all()
    c = q.float().double()
    assert c.abs().max() <= TOP[dtype]
    if dtype == "i8":
        step = torch.ones_like(c)
    else:
        step = 2.0 ** (torch.floor(torch.log2((want / s[:, None]).abs().clamp_min(2.0 ** -6))) - 3)
    err = (c * s[:, None] - want).abs()
    assert (err <= (0.5 + 2.0 ** -10) * step * s[:, None] + 2.0 ** -17 * mag).all(), float(err.max())


# ------------------------------------------------------------------------------------- quantize

def run_quantize(x, q, scale, xd, qd, stream=0):
    api.quantize_rows(x.shape[0], x.shape[1], ptr(x), DT[xd], ptr(q), DT[qd], ptr(scale), ld_x=x.stride(0),
                      ld_q=q.stride(0), stream=stream)


@pytest.mark.parametrize("h", [1, 7, 64, 255, 256, 512, 768, 1152, 1500, 1543, 1790, 2056, 3000, 4096, 5000, 6101, 8000,
                               8200, 12000, 20000, 32761, 32768])
@pytest.mark.parametrize("xd,qd", [("f16", "i8"), ("bf16", "e4m3"), ("f32", "i8"), ("f32", "e4m3")])
def test_quantize_rows(h, xd, qd):
    for m, pad, off in ((1, 0, 0), (5, 0, 0), (67, 8, 8), (33, 3, 1)):
        x = filled(rows_of(m, h, h + m), xd, pad, off)
        q = buffer(m, h, qd, pad, off, fill=0x55)
        scale = torch.full((m,), float("nan"), device="cuda")
        run_quantize(x, q, scale, xd, qd)
        check_codes(q, scale, x, qd)


@pytest.mark.parametrize("qd", ["i8", "e4m3"])
@pytest.mark.parametrize("h", [8, 768, 771, 5000])
def test_quantize_edge_rows(h, qd):
    """Zeros, the smallest and largest magnitudes, a NaN, infinities: each row alone."""
    x = rows_of(9, h, 3)
    x[0] = 0
    x[1] = 1e-38
    x[2] = 0
    x[2, h // 2] = 3e38
    x[3, h - 1] = float("nan")
    x[4, 0] = float("inf")
    x[5, h // 3] = float("-inf")
    x[6] = -0.0
    x[7] = 2.0 ** -126
    q, scale = buffer(9, h, qd), torch.empty(9, device="cuda")
    run_quantize(x, q, scale, "f32", qd)
    ok = [0, 1, 2, 6, 7, 8]
    check_codes(q[ok], scale[ok], x[ok], qd)
    assert (q[0].float() == 0).all() and scale[0] == FLOOR
    v = q.float() * scale[:, None]
    assert torch.isnan(v[3]).all() and torch.isnan(v[4]).all() and torch.isnan(v[5]).all()


def test_rounding_is_to_nearest_even():
    """A row whose largest magnitude is `top` has scale 1, so its codes are its values rounded."""
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 0.49999997, 63.5]], device="cuda")
    q, s = buffer(1, 8, "i8"), torch.empty(1, device="cuda")
    run_quantize(x, q, s, "f32", "i8")
    assert s.item() == 1.0 and q.cpu().tolist() == [[127, 0, 2, 2, 0, -2, 0, 64]]
    x = torch.tensor([[448.0, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, -17.0, 416.0, 432.0]], device="cuda")
    q = buffer(1, 8, "e4m3")
    run_quantize(x, q, s, "f32", "e4m3")
    assert s.item() == 1.0
    assert q.float().cpu().tolist() == [[448.0, 16.0, 20.0, 0.0, 2.0 ** -8, -16.0, 416.0, 448.0]]


@pytest.mark.parametrize("qd", ["i8", "e4m3"])
@pytest.mark.parametrize("h,pad", [(64, 0), (768, 0), (771, 0), (2048, 0), (1001, 3)])
def test_exact_ties_of_16_bit_rows(h, pad, qd):
    """f16 rows whose largest value is a power of two times `top`: every quotient v / scale is exact, many
    fall halfway between two codes, and all must go to the even one."""
    m = 64
    g = torch.Generator(device="cuda")
    g.manual_seed(h)
    v = torch.randint(-254, 255, (m, h), generator=g, device="cuda").float() / 2  # halves, within +-127
    if qd == "e4m3":
        v = torch.round(v * 8) / 4  # quarters and coarser: ties of every binade
    top = TOP[qd]
    v = v.clamp(-top, top)
    v[:, h // 2] = top
    up = torch.arange(m, device="cuda")[:, None] % 5 - 2
    x = filled(v * 2.0 ** up, "f32" if qd == "e4m3" else "f16", pad)
    q, s = buffer(m, h, qd, pad), torch.empty(m, device="cuda")
    run_quantize(x, q, s, "f32" if qd == "e4m3" else "f16", qd)
    assert torch.equal(s, 2.0 ** up[:, 0].float())
    want = torch.round(v) if qd == "i8" else v.to(torch.float8_e4m3fn).float()  # both to the even one
    assert torch.equal(q.float(), want)


# ------------------------------------------------------------------------------------- norm

def norm_want(x, res, post, gain, scalar):
    def rms(v):
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)
    x = x.double()
    xt = x if post is None else rms(x) * post.double()
    r = torch.zeros_like(x) if res is None else res.double()
    h = (r + xt) * scalar
    n = rms(h) if gain is None else rms(h) * gain.double()
    mag = (r.abs() + xt.abs()) * abs(scalar)
    return h, n, mag, mag * (n.abs().amax(1, keepdim=True) / (h * (1 if gain is None else gain)).abs().amax(1, keepdim=True)
                             .clamp_min(1e-300)) * (1 if gain is None else gain.abs())


@pytest.mark.parametrize("h", [1, 5, 64, 117, 256, 512, 768, 1024, 1152, 1543, 2048, 2568, 4096, 5000, 6000, 8000, 9001,
                               12000, 16384, 20004, 32761, 32768])
@pytest.mark.parametrize("xd,hd,qd", [("f16", "bf16", "i8"), ("bf16", "bf16", "e4m3"), ("f32", "f32", "i8"),
                                      ("f16", "f32", "e4m3"), ("f32", "f16", "e4m3")])
def test_norm_residual_q8(h, xd, hd, qd):
    for m, pad, off, post_on, res_on, gain_on, scalar in ((1, 0, 0, True, True, True, 1.0),
                                                          (66, 0, 0, False, True, True, 0.75),
                                                          (35, 8, 8, True, True, True, 1.5),
                                                          (19, 5, 3, True, False, True, 1.0),
                                                          (17, 8, 0, False, True, False, 1.0)):
        x = filled(rows_of(m, h, h + m, 0.5), xd, pad, off)
        res = filled(2 * rows_of(m, h, h + m + 1, 0.5), hd, pad, off) if res_on else None
        g = torch.Generator(device="cuda")
        g.manual_seed(h)
        gains = torch.randn(2 * h + 8, generator=g, device="cuda") * 0.2 + 1
        o = 1 if off % 4 else 0  # gains off a 16-byte boundary with the odd layouts
        post = gains[o:o + h] if post_on else None
        gain = gains[h + 1 + o:h + 1 + o + h] if gain_on and o else (gains[h + (-h) % 4:][:h] if gain_on else None)
        hout = buffer(m, h, hd, pad, off)
        q = buffer(m, h, qd, pad, off)
        scale = torch.empty(m, device="cuda")
        api.norm_residual_q8(m, h, ptr(x), DT[xd], ptr(q), DT[qd], ptr(scale), gain=ptr(gain), post_gain=ptr(post),
                             residual=ptr(res), h=ptr(hout), h_dtype=DT[hd], eps=EPS, layer_scalar=scalar,
                             ld_x=x.stride(0), ld_residual=res.stride(0) if res_on else 0, ld_h=hout.stride(0),
                             ld_q=q.stride(0))
        h_want, n_want, mag, n_mag = norm_want(x, res, post, gain, scalar)
        err = (hout.double() - h_want).abs()
        assert (err <= U[hd] * h_want.abs() + 2.0 ** -18 * mag + TINY[hd]).all(), (m, float(err.max()))
        check_codes(q, scale, n_want, qd, n_mag)


@pytest.mark.parametrize("h", [768, 771, 2048, 2051, 9001])
def test_norm_in_place_and_without_h(h):
    m = 37
    x, res = filled(rows_of(m, h, 1), "f16"), filled(rows_of(m, h, 2), "bf16")
    gain = rows_of(1, h, 3, 0.0)[0] * 0.1 + 1
    outs = []
    for mode in ("apart", "in place", "none"):
        r = res.clone()
        hout = {"apart": torch.empty_like(r), "in place": r, "none": None}[mode]
        q, s = buffer(m, h, "i8"), torch.empty(m, device="cuda")
        api.norm_residual_q8(m, h, ptr(x), DT["f16"], ptr(q), DT["i8"], ptr(s), gain=ptr(gain), residual=ptr(r),
                             h=ptr(hout), h_dtype=DT["bf16"], eps=EPS)
        outs.append((q.clone(), s, hout))
    assert torch.equal(outs[0][2], outs[1][2])
    for q, s, _ in outs[1:]:
        assert torch.equal(q, outs[0][0]) and torch.equal(s, outs[0][1])


@pytest.mark.parametrize("h", [768, 771])
def test_norm_edge_rows(h):
    """A zero row (x and residual), one that holds a NaN, one an infinity: the others are untouched."""
    x, res = filled(rows_of(6, h, 1), "f16"), filled(rows_of(6, h, 2), "bf16")
    x[0] = 0
    res[0] = 0
    x[2, h - 1] = float("nan")
    res[3, 0] = float("inf")
    clean = [0, 1, 4, 5]
    hout, q, s = torch.empty_like(res), buffer(6, h, "e4m3"), torch.empty(6, device="cuda")
    api.norm_residual_q8(6, h, ptr(x), DT["f16"], ptr(q), DT["e4m3"], ptr(s), residual=ptr(res), h=ptr(hout),
                         h_dtype=DT["bf16"], eps=EPS)
    _, n, _, n_mag = norm_want(x[clean], res[clean], None, None, 1.0)
    check_codes(q[clean], s[clean], n, "e4m3", n_mag)
    assert (q[0].float() == 0).all() and s[0] == FLOOR
    assert torch.isnan(q.float() * s[:, None])[[2, 3]].all()


@pytest.mark.parametrize("qd", ["i8", "e4m3"])
@pytest.mark.parametrize("h", [64, 77, 768, 2051])
@pytest.mark.parametrize("eps", [1e-30, 1e-6, 1.0])
def test_norm_zero_rows_whatever_the_eps(h, qd, eps):
    x = torch.zeros((5, h), dtype=torch.float32, device="cuda")
    x[1] = 1.0
    q, s = buffer(5, h, qd), torch.empty(5, device="cuda")
    api.norm_residual_q8(5, h, ptr(x), DT["f32"], ptr(q), DT[qd], ptr(s), h_dtype=DT["f32"], eps=eps)
    rows = [0, 2, 3, 4]
    assert (q[rows].float() == 0).all() and (s[rows] == FLOOR).all()
    assert (q[1].float() == TOP[qd]).all()


def test_rows_past_32_bit_offsets():
    """Element offsets past 2^31: the last rows of a 70,000 x 32,768 matrix."""
    m, h = 70000, 32768
    x = torch.zeros((m, h), dtype=torch.float16, device="cuda")
    x[-3:] = rows_of(3, h, 5).half()
    q, s = torch.empty((m, h), dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    run_quantize(x, q, s, "f16", "i8")
    check_codes(q[-3:], s[-3:], x[-3:], "i8")
    assert (s[:-3] == FLOOR).all() and not q[: 1000].any() and not q[-1003:-3].any()


# ------------------------------------------------------------------------------------- linear

def act64(v, kind):
    if kind == "relu":
        return v.clamp_min(0)
    if kind == "silu":
        return v * torch.sigmoid(v)
    if kind == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))  # 0.5 v (1 + tanh z)
    if kind == "gelu_erf":
        return 0.5 * v * torch.special.erfc(-math.sqrt(0.5) * v)
    return v


class Case:
    """One product: operands with pitches and offsets, everything the epilogue takes, 64-bit values."""

    def __init__(self, m, n, k, dtype, out, act="none", gated=False, bias=False, res=False, scales=None, seed=0,
                 pad=None, off=0, ypad=0, yoff=0):
        size = 1 if dtype in ("i8", "e4m3") else 2
        pad = (-k) % (16 // size) if pad is None else pad
        self.m, self.n, self.k, self.dtype, self.out, self.act = m, n, k, dtype, out, act

        def operand(rows, std, seed):
            v = rows_of(rows, k, seed, 0.3) * std
            if dtype == "i8":
                v = (v * 40 / std).round().clamp(-127, 127)
            elif dtype == "e4m3":
                v = (v * 60 / std).clamp(-448, 448)
            return filled(v, dtype, pad, off)

        self.x, self.w = operand(m, 0.7, seed), operand(n, 1.5 / math.sqrt(k), seed + 1)
        self.wu = operand(n, 1.5 / math.sqrt(k), seed + 2) if gated else None
        scales = size == 1 if scales is None else scales
        sx = 0.7 / 40 if dtype == "i8" else (0.7 / 60 if dtype == "e4m3" else 1.0)
        sw = sx / 0.7 * 1.5 / math.sqrt(k) if size == 1 else 1.0
        self.xs = (1 + 0.3 * torch.rand(m, device="cuda")) * sx if scales else None
        self.ws = (1 + 0.3 * torch.rand(n, device="cuda")) * sw if scales else None
        self.wus = (1 + 0.3 * torch.rand(n, device="cuda")) * sw if scales and gated else None
        self.b = torch.randn(n, device="cuda") if bias else None
        self.bu = torch.randn(n, device="cuda") if bias and gated else None
        self.res = filled(rows_of(m, n, seed + 3, 0.0), out, ypad, yoff) if res else None
        self.y = buffer(m, n, out, ypad, yoff, fill=float("nan"))

    def run(self, stream=0, y=None):
        y = self.y if y is None else y
        api.linear(self.m, self.n, self.k, DT[self.dtype], ptr(self.x), ptr(self.w), ptr(y), DT[self.out],
                   x_scale=ptr(self.xs), w_scale=ptr(self.ws), w_up=ptr(self.wu), w_up_scale=ptr(self.wus),
                   bias=ptr(self.b), bias_up=ptr(self.bu), activation=api.ACTIVATIONS[self.act], residual=ptr(self.res),
                   ldx=self.x.stride(0), ldw=self.w.stride(0), ld_residual=self.res.stride(0) if self.res is not None else 0,
                   ldy=y.stride(0), stream=stream)
        return y

    def want(self, rows=slice(None)):
        def product(w, ws, b):
            x64, w64 = self.x[rows].float().double(), w.float().double()
            v, mag = x64 @ w64.T, x64.abs() @ w64.abs().T
            s = 1.0
            if self.xs is not None:
                s = self.xs[rows].double()[:, None] * ws.double()
            err = mag * s * (2.0 ** -22 if self.dtype == "i8" else (self.k + 8) * 2.0 ** -23) + (v * s).abs() * 2.0 ** -21
            v = v * s
            if b is not None:
                v, err = v + b.double(), err + (v.abs() + b.abs()) * 2.0 ** -23
            return v, err

        v, err = product(self.w, self.ws, self.b)
        y = act64(v, self.act)
        if self.act != "none":
            err = 1.2 * err + 2.0 ** -15 * y.abs() + 1e-30
        if self.wu is not None:
            u, eu = product(self.wu, self.wus, self.bu)
            y, err = y * u, err * u.abs() + eu * y.abs() + err * eu
        if self.res is not None:
            y, err = y + self.res[rows].double(), err + (y.abs() + self.res[rows].double().abs()) * 2.0 ** -23
        return y, err + U[self.out] * y.abs() + TINY[self.out]

    def check(self, rows=slice(None)):
        y, bound = self.want(rows)
        err = (self.y[rows].double() - y).abs()
        bad = ~(err <= bound)
        assert not bad.any(), (int(bad.sum()), [int(i) for i in bad.nonzero()[0]], float((err / bound).nan_to_num(9e9).max()))


SIZES = [(1, 1, 1), (1, 768, 768), (2, 100, 64), (3, 129, 72), (5, 1543, 200), (8, 256, 1152), (9, 64, 40),
         (16, 513, 257), (17, 768, 128), (31, 80, 1000), (33, 257, 130), (64, 768, 768), (65, 200, 96), (100, 1000, 64),
         (128, 256, 256), (129, 384, 333), (200, 72, 4100), (256, 512, 64), (300, 1152, 768), (513, 257, 129),
         (1000, 100, 31), (1500, 768, 1152), (4100, 264, 72)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype,out", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("i8", "f16"), ("i8", "f32"),
                                       ("e4m3", "bf16"), ("e4m3", "f32")])
def test_linear_sizes(m, n, k, dtype, out):
    c = Case(m, n, k, dtype, out, seed=m + n + k)
    c.run()
    c.check()
    c = Case(m, n, k, dtype, out, act="gelu_tanh", bias=True, res=True, seed=m + n + k + 7, ypad=(-n) % 8)
    c.run()
    c.check()
    c = Case(m, n, k, dtype, out, act="silu", gated=True, bias=True, res=(m % 2 == 1), seed=m + n + k + 9)
    c.run()
    c.check()


@pytest.mark.parametrize("m,n,k", [(3, 2500, 300), (16, 2376, 72), (20, 2400, 80), (32, 1300, 200), (40, 2400, 100),
                                   (64, 96, 1000), (33, 4100, 1040), (20, 7300, 700)])
@pytest.mark.parametrize("dtype,out", [("f16", "f32"), ("bf16", "f16"), ("i8", "f32"), ("e4m3", "bf16")])
def test_linear_few_rows_of_many_columns(m, n, k, dtype, out):
    """Either side of the rules that choose how many rows of w a block of the few-rows kernel takes, and
    between it and the tensor-memory kernel."""
    for gated in (False, True):
        c = Case(m, n, k, dtype, out, act="gelu_erf", gated=gated, bias=True, res=True, seed=m + n)
        c.run()
        c.check()


@pytest.mark.parametrize("m,n,k", [(100, 300, 3000), (65, 2049, 2100), (128, 64, 8100), (257, 777, 1600), (130, 61, 2056),
                                   (500, 520, 2064)])
@pytest.mark.parametrize("dtype,out", [("f16", "f16"), ("bf16", "f32"), ("i8", "f32"), ("e4m3", "bf16")])
def test_linear_split_over_k(m, n, k, dtype, out):
    """Few tiles and a long K: clusters of 2, 4 and 8 CTAs share a tile's K steps."""
    for act, gated, bias, res in (("none", False, False, False), ("gelu_tanh", False, True, True), ("silu", True, True, True)):
        c = Case(m, n, k, dtype, out, act=act, gated=gated, bias=bias, res=res, seed=m + k, ypad=(3 if gated else 0))
        c.run()
        c.check()
        again = torch.empty_like(c.y)
        again.copy_(c.y)
        c.run()
        assert torch.equal(again, c.y)


@pytest.mark.parametrize("dtype,k", [("f16", 1000), ("bf16", 1056), ("i8", 2100), ("e4m3", 2064)])
@pytest.mark.parametrize("n,ypad,yoff", [(520, 0, 0), (777, 0, 0), (777, 7, 0), (520, 3, 5), (264, 8, 8)])
def test_linear_on_pairs(dtype, k, n, ypad, yoff):
    """Products of enough 256 x 256 tiles for the CTA-pair kernel: several tiles per pair, ragged last
    tiles, outputs on and off 16-byte rows, each epilogue's warps."""
    for m, act, gated, res, out in ((20011, "none", False, True, "bf16"), (20011, "gelu_erf", False, True, "f16"),
                                    (16384, "silu", True, True, "f16"), (20011, "relu", False, True, "f32"),
                                    (19999, "gelu_tanh", True, False, "f32"), (16385, "none", False, False, "f16")):
        c = Case(m, n, k, dtype, out, act=act, gated=gated, bias=True, res=res, seed=n + k, ypad=ypad, yoff=yoff)
        c.run()
        c.check()


@pytest.mark.parametrize("m,n,k", [(4, 200, 320), (70, 200, 320), (700, 520, 192)])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu_tanh", "gelu_erf"])
@pytest.mark.parametrize("gated,bias,res", [(False, True, True), (True, False, False), (True, True, True)])
def test_linear_epilogues(m, n, k, act, gated, bias, res):
    for dtype, out in (("f16", "f16"), ("e4m3", "f32"), ("i8", "bf16")):
        c = Case(m, n, k, dtype, out, act=act, gated=gated, bias=bias, res=res, seed=m + n)
        c.run()
        c.check()


@pytest.mark.parametrize("m", [3, 50, 400])
@pytest.mark.parametrize("dtype,pad,off", [("f16", 1, 0), ("f16", 8, 3), ("bf16", 0, 8), ("i8", 5, 0), ("e4m3", 16, 7),
                                           ("i8", 16, 16)])
@pytest.mark.parametrize("ypad,yoff", [(0, 0), (3, 1), (8, 8), (1, 0)])
def test_linear_pitches_and_alignments(m, dtype, pad, off, ypad, yoff):
    c = Case(m, 203, 176, dtype, "f16", act="gelu_erf", bias=True, res=True, pad=pad, off=off, ypad=ypad, yoff=yoff,
             gated=True, seed=m)
    whole = torch.as_strided(c.y, (c.m, c.y.stride(0)), (c.y.stride(0), 1))
    before = whole[:, c.n:].clone()
    c.run()
    c.check()
    assert torch.equal(whole[:, c.n:].isnan(), before.isnan())  # nothing is written between the rows


@pytest.mark.parametrize("m,n,k", [(3, 77, 100), (64, 128, 300), (600, 300, 1000), (1024, 512, 4096)])
def test_linear_int8_sums_are_exact(m, n, k):
    """All codes at +-127 too: sums past 2^24, rounded once to f32."""
    c = Case(m, n, k, "i8", "f32", scales=False, seed=1)
    c.x[: m // 2] = 127
    c.w[: n // 2] = torch.where(torch.arange(k, device="cuda") % 7 == 0, -127, 127).to(torch.int8)
    c.run()
    want = (c.x.double() @ c.w.double().T).float()
    assert torch.equal(c.y, want)


@pytest.mark.parametrize("m", [2, 40, 300])
def test_linear_in_place_residual(m):
    c = Case(m, 264, 128, "f16", "bf16", bias=True, res=True, seed=4)
    apart = c.run().clone()
    c.check()
    c.run(y=c.res)
    assert torch.equal(c.res, apart)


@pytest.mark.parametrize("m", [2, 40, 300, 2000])
@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
def test_linear_non_finite_stay_in_their_rows(m, dtype):
    """A NaN in one row of x, an infinity (f16) in one row of w: that row and that column only."""
    c = Case(m, 200, 96, dtype, "f32", act="gelu_tanh", seed=6)
    x = c.x.float()
    x[1, 95] = float("nan")
    c.x.copy_(x.to(c.x.dtype))
    if dtype == "f16":
        c.w[7, 3] = float("inf")
    c.run()
    fine = torch.isfinite(c.y)
    ok = torch.ones_like(fine)
    ok[1] = False
    assert torch.isnan(c.y[1]).all()
    if dtype == "f16":
        ok[:, 7] = False
    assert fine[ok].all()


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "gelu_erf", "relu", "none"])
@pytest.mark.parametrize("m", [1, 64, 300])
def test_activation_over_its_range(act, m):
    """x w^T with one column of K: the activation of chosen values, out to where it is 0 or v."""
    v = torch.linspace(-100, 100, 1023, device="cuda").half()
    v = torch.cat([v, torch.tensor([0.0, -0.0, 65504.0, -65504.0, 1e-4, -1e-4, -5.5], device="cuda").half()])
    n = v.numel()
    c = Case(m, n, 1, "f16", "f32", act=act, seed=1)
    c.w[:, 0] = v
    c.x[:, 0] = 1.0
    c.run()
    want = act64(v.double(), act).expand(m, n)
    assert ((c.y.double() - want).abs() <= 2.0 ** -15 * want.abs() + 1e-30).all()


def test_linear_runs_on_the_given_stream_and_repeats():
    c = Case(1000, 768, 768, "f16", "f16", act="silu", bias=True, res=True, seed=8)
    small = Case(2, 768, 768, "i8", "f32", seed=9)
    first, first_small = c.run().clone(), small.run().clone()
    st = torch.cuda.Stream()
    x = c.x.clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        c.x.zero_()
        torch.cuda._sleep(2_000_000)
        c.x.copy_(x)
        c.y.fill_(0)
        small.y.fill_(0)
        c.run(stream=st.cuda_stream)
        small.run(stream=st.cuda_stream)
    st.synchronize()
    assert torch.equal(c.y, first) and torch.equal(small.y, first_small)


def test_linear_graph_capture():
    """Captured calls replay on new inputs in the same buffers."""
    cases = [Case(m, 768, 768, d, "f16", act="gelu_tanh", bias=True, res=True, seed=m)
             for m, d in ((1, "f16"), (40, "i8"), (900, "e4m3"))]
    st = torch.cuda.Stream()
    for c in cases:
        c.run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        for c in cases:
            c.run(stream=st.cuda_stream)
    for c in cases:
        c.x.copy_(filled(torch.flip(c.x.float(), [0, 1]), c.dtype))
        c.y.fill_(0)
    g.replay()
    torch.cuda.synchronize()
    for c in cases:
        c.check()


def test_linear_output_past_32_bit_offsets():
    """2,100,000 x 1,032 outputs: element offsets past 2^31."""
    c = Case(2_100_000, 1032, 16, "f16", "f16", seed=2)
    c.run()
    c.check(slice(-70, None))
    c.check(slice(0, 70))


@pytest.mark.parametrize("m,n", [(540_000, 24), (3, 540_000), (300, 540_000)])
def test_linear_operands_past_32_bit_offsets(m, n):
    """x or w of more than 2^31 elements: each kernel's last rows and columns."""
    k = 4000
    c = Case.__new__(Case)
    c.m, c.n, c.k, c.dtype, c.out, c.act = m, n, k, "i8", "f32", "none"
    c.x = torch.zeros((m, k), dtype=torch.int8, device="cuda")
    c.w = torch.zeros((n, k), dtype=torch.int8, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(m + n)
    for t in (c.x, c.w):
        tail = t[-2000:]
        tail.copy_(torch.randint(-127, 128, tail.shape, generator=g, device="cuda", dtype=torch.int8))
    c.xs = c.ws = c.wus = c.wu = c.b = c.bu = c.res = None
    c.y = torch.full((m, n), float("nan"), device="cuda")
    c.run()
    want = (c.x[-2000:].double() @ c.w[-2000:].double().T).float()
    assert torch.equal(c.y[-2000:, -2000:], want)
    assert not c.y.isnan().any()


def test_zero_rows_are_a_no_op():
    api.linear(0, 8, 8, DT["f16"], 0, 0, 0, DT["f16"])
    api.quantize_rows(0, 8, 0, DT["f16"], 0, DT["i8"], 0)
    api.norm_residual_q8(0, 8, 0, DT["f16"], 0, DT["i8"], 0)


def test_operators_together():
    """An int8 feed-forward half of a layer: what the four calls give against the same steps in 64 bits
    on the codes and scales that came out (each step is held to its own bound by the tests above)."""
    m, h, f = 300, 768, 1152
    x, res = filled(rows_of(m, h, 1, 0.3), "f16"), filled(rows_of(m, h, 2, 0.3), "bf16")
    post = torch.rand(h, device="cuda") + 0.5
    gain = torch.rand(h, device="cuda") + 0.5
    ws = []
    for i, (n, k) in enumerate(((f, h), (f, h), (h, f))):
        w = rows_of(n, k, 10 + i, 0.2) / math.sqrt(k)
        q, s = buffer(n, k, "i8"), torch.empty(n, device="cuda")
        run_quantize(w, q, s, "f32", "i8")
        ws.append((q, s, w))
    q, s = buffer(m, h, "i8"), torch.empty(m, device="cuda")
    hout, a, y = torch.empty_like(res), buffer(m, f, "f16"), buffer(m, h, "f16")
    api.norm_residual_q8(m, h, ptr(x), DT["f16"], ptr(q), DT["i8"], ptr(s), gain=ptr(gain), post_gain=ptr(post),
                         residual=ptr(res), h=ptr(hout), h_dtype=DT["bf16"])
    api.linear(m, f, h, DT["i8"], ptr(q), ptr(ws[0][0]), ptr(a), DT["f16"], x_scale=ptr(s), w_scale=ptr(ws[0][1]),
               w_up=ptr(ws[1][0]), w_up_scale=ptr(ws[1][1]), activation=api.ACTIVATIONS["gelu_tanh"])
    qa, sa = buffer(m, f, "i8"), torch.empty(m, device="cuda")
    run_quantize(a, qa, sa, "f16", "i8")
    api.linear(m, h, f, DT["i8"], ptr(qa), ptr(ws[2][0]), ptr(y), DT["f16"], x_scale=ptr(sa), w_scale=ptr(ws[2][1]))
    _, n64, _, _ = norm_want(x, res, post, gain, 1.0)
    a64 = act64(n64 @ ws[0][2].double().T, "gelu_tanh") * (n64 @ ws[1][2].double().T)
    y64 = a64 @ ws[2][2].double().T
    # 8 bits with a row's largest value at 127: each quantisation adds about max / (127 sqrt(12)) of
    # noise per value, under 1.2 % of the row's rms for maxima of up to 5 rms; five of them
    # (three weights, two activations; gate and up both enter a) stay under 4 % in the 2-norm
    assert float((y.double() - y64).norm() / y64.norm()) < 0.04


def test_the_example_runs():
    """examples/int8_feed_forward.py end to end: the same noise bound as above."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "int8_feed_forward.py")
    spec = importlib.util.spec_from_file_location("int8_feed_forward", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    err, cos = example.main(["--tokens", "333"])
    assert err < 0.04 and cos > 0.998
