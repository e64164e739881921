"""The int8 feed-forward half of examples/int8_feed_forward.py: nothing between its two products is held in fewer
than 32 bits but the codes."""
from __future__ import annotations

import importlib.util
import os

import pytest

from glypr_b200 import api

from .conftest import ROOT

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def half(h, f, m, seed, up=1.0, down=1.0):
    """The example's class on random weights, its inputs and its output."""
    spec = importlib.util.spec_from_file_location("int8_feed_forward", os.path.join(ROOT, "examples", "int8_feed_forward.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    api.load_library()
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")
    w = [randn(f, h) / h ** 0.5 * up, randn(f, h) / h ** 0.5 * up, randn(h, f) / f ** 0.5 * down]
    ffn = example.Int8FeedForward(*w, 1 + 0.1 * randn(h), 1 + 0.1 * randn(h), m)
    attn, residual = randn(m, h).half(), (3 * randn(m, h)).bfloat16()
    y = torch.empty((m, h), dtype=torch.float16, device="cuda")
    ffn(attn, residual, y)
    return ffn, y


def want(ffn):
    """y in 64 bits from the codes and scales that the norm wrote."""
    def value(codes, scale):
        return codes.double() * scale.double()[:, None]
    n = value(ffn.q, ffn.scales[0])
    gate, up, down = (value(*w) for w in (ffn.gate, ffn.up, ffn.down))
    v = n @ gate.T
    a = v * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3)) * (n @ up.T)
    s = a.abs().amax(1) / 127
    return a, value(torch.round(a / s[:, None]), s) @ down.T


def test_codes_are_those_of_the_unrounded_product():
    """f16's rounding of y (2^-11 at most), and codes that the activation's error of about 1e-6 moves over a
    rounding boundary: of values of ten steps or so one in 1e5, each off by a step, a fifteenth of the rms:
    2e-4 in all.  A rounding of `a` to f16 moves a hundred times as many (2.7e-3)."""
    ffn, y = half(768, 1152, 600, 1)
    _, y64 = want(ffn)
    assert float((y.double() - y64).norm() / y64.norm()) < 1e-3


def test_products_beyond_f16_stay_finite():
    ffn, y = half(256, 512, 70, 2, up=300.0, down=1e-4)
    a, y64 = want(ffn)
    assert float(a.abs().max()) > 65504 * 2
    assert torch.isfinite(y).all()
    assert float((y.double() - y64).norm() / y64.norm()) < 1e-3
