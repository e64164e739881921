"""Argument checks of glp_norm_residual_q8, glp_quantize_rows and glp_linear: each refusal comes with
GLP_ERR_INVALID_ARG and a message before any CUDA call, so it needs no GPU (the addresses below are
never touched)."""
from __future__ import annotations

import pytest

from glypr_b200 import api

DT = api.DTYPES
P = 1 << 20  # a stand-in address, 16-byte aligned


def refused(call, word):
    with pytest.raises(api.GlyprError) as e:
        call()
    assert e.value.code == api.GLP_ERR_INVALID_ARG
    assert word in e.value.message, e.value.message


def linear(m=4, n=8, k=16, dtype="f16", x=P, w=P, y=P, out="f16", **kw):
    return lambda: api.linear(m, n, k, DT.get(dtype, dtype), x, w, y, DT.get(out, out), **kw)


@pytest.mark.parametrize("call,word", [
    (linear(m=-1), "M >= 0"), (linear(n=0), "N >= 1"), (linear(k=0), "K >= 1"),
    (linear(dtype="f32"), "operands"), (linear(dtype=9), "operands"), (linear(dtype=-1), "operands"),
    (linear(out="i8"), "y must be"), (linear(out="e4m3"), "y must be"), (linear(out=7), "y must be"),
    (linear(activation=5), "activation"), (linear(activation=-1), "activation"),
    (linear(dtype="i8", k=131072), "131071"), (linear(m=2 ** 30 + 1), "2^30"), (linear(n=2 ** 30 + 1), "2^30"),
    (linear(k=2 ** 28 + 1), "2^28"),
    (linear(x=0), "null"), (linear(w=0), "null"), (linear(y=0), "null"),
    (linear(ldx=15), "shorter than K"), (linear(ldw=15), "shorter than K"), (linear(ldx=-16), "shorter than K"),
    (linear(ldy=7), "shorter than N"), (linear(residual=P, ld_residual=7), "shorter than N"),
    (linear(residual=P, ldy=8, ld_residual=16), "same row pitch"),
    (linear(bias_up=P), "need w_up"), (linear(w_up_scale=P), "need w_up"),
    (linear(x=P + 1), "aligned"), (linear(out="f32", y=P + 2), "aligned"), (linear(bias=P + 2), "aligned"),
    (linear(x_scale=P + 1), "aligned"), (linear(w_up=P + 1), "aligned"), (linear(residual=P + 1), "aligned"),
])
def test_linear_refusals(call, word):
    refused(call, word)


def quantize(m=4, h=16, x=P, xd="f16", q=P, qd="i8", s=P, **kw):
    return lambda: api.quantize_rows(m, h, x, DT.get(xd, xd), q, DT.get(qd, qd), s, **kw)


def norm(m=4, h=16, x=P, xd="f16", q=P, qd="i8", s=P, hd="bf16", **kw):
    return lambda: api.norm_residual_q8(m, h, x, DT.get(xd, xd), q, DT.get(qd, qd), s, h_dtype=DT.get(hd, hd), **kw)


@pytest.mark.parametrize("make", [quantize, norm])
@pytest.mark.parametrize("kw,word", [
    ({"m": -1}, "M >= 0"), ({"h": 0}, "H <= 32768"), ({"h": 32769}, "H <= 32768"), ({"xd": "i8"}, "F32"),
    ({"xd": 5}, "F32"), ({"qd": "f16"}, "I8 or E4M3"), ({"qd": -1}, "I8 or E4M3"), ({"x": 0}, "null"),
    ({"q": 0}, "null"), ({"s": 0}, "null"), ({"ld_x": 15}, "shorter than H"), ({"ld_q": 8}, "shorter than H"),
    ({"x": P + 1}, "aligned"), ({"s": P + 2}, "aligned"),
])
def test_row_refusals(make, kw, word):
    refused(make(**kw), word)


@pytest.mark.parametrize("kw,word", [
    ({"hd": "i8"}, "F32"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"),
    ({"residual": P, "ld_residual": 3}, "shorter than H"), ({"h_out": P, "ld_h": 3}, "shorter than H"),
    ({"residual": P, "h_out": P, "ld_h": 24}, "same row pitch"), ({"gain": P + 2}, "aligned"),
    ({"post_gain": P + 1}, "aligned"), ({"residual": P + 1}, "aligned"), ({"h_out": P + 1}, "aligned"),
])
def test_norm_refusals(kw, word):
    kw = {("h" if k == "h_out" else k): v for k, v in kw.items()}
    hl = kw.pop("h", 0)
    refused(lambda: api.norm_residual_q8(4, 16, P, DT["f16"], P, DT["i8"], P, h=hl,
                                         h_dtype=DT.get(kw.get("hd", "bf16")),
                                         **{k: v for k, v in kw.items() if k != "hd"}), word)


def test_null_argument_blocks():
    lib = api.load_library()
    assert lib.glp_linear(None, None) == api.GLP_ERR_INVALID_ARG
    assert lib.glp_norm_residual_q8(None, None) == api.GLP_ERR_INVALID_ARG
    assert b"NULL" in lib.glp_last_error()
