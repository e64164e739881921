"""The feed-forward half of an encoder layer in int8, from Q8_0 weights.

    python examples/int8_feed_forward.py [--tokens N]

Takes a layer's gate, up and down weights as a GGUF holds them (Q8_0 blocks; here random ones of 768 and
1,152 columns), turns each weight row into int8 codes with one scale (glp_q8_0_dequant, then
glp_quantize_rows, once), and runs

    h, (q, s)  = glp_norm_residual_q8     h += post-norm of the attention block's output; pre-norm in int8
    a          = glp_linear (gated)       gelu_tanh(q Wgate^T) * (q Wup^T), f32: in f16 its
                                          rounding would move codes, and 65,504 end it
    (qa, sa)   = glp_quantize_rows        a in int8
    y          = glp_linear               qa Wdown^T, f16: the input of the layer's next post-norm

on N rows of residual stream, against the same half in f32 on the Q8_0 weights' exact values.  PyTorch
holds the device memory; the operators take its pointers.
"""
from __future__ import annotations

import argparse
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

import numpy as np  # noqa: E402
import torch  # noqa: E402

from glypr_b200 import api, synth  # noqa: E402

DT = api.DTYPES
EPS = 1e-6


class Int8FeedForward:
    """One layer's feed-forward half: int8 weights with a scale per row, workspaces for up to max_tokens."""

    def __init__(self, gate, up, down, post_attn_gain, pre_ffn_gain, max_tokens):
        self.h, self.f = gate.shape[1], gate.shape[0]
        self.post_gain, self.gain = post_attn_gain, pre_ffn_gain
        self.gate, self.up, self.down = (self.quantized(w) for w in (gate, up, down))
        dev = gate.device
        self.q = torch.empty((max_tokens, self.h), dtype=torch.int8, device=dev)
        self.a = torch.empty((max_tokens, self.f), device=dev)
        self.qa = torch.empty((max_tokens, self.f), dtype=torch.int8, device=dev)
        self.scales = torch.empty((2, max_tokens), device=dev)

    @staticmethod
    def quantized(w):
        """f32 rows -> (int8 codes, one scale per row)."""
        q, s = torch.empty(w.shape, dtype=torch.int8, device=w.device), torch.empty(w.shape[0], device=w.device)
        api.quantize_rows(w.shape[0], w.shape[1], w.data_ptr(), DT["f32"], q.data_ptr(), DT["i8"], s.data_ptr(),
                          stream=torch.cuda.current_stream().cuda_stream)
        return q, s

    def __call__(self, attn_out, residual, y):
        """attn_out f16 [m, h] (the O projection), residual bf16 [m, h] (updated in place) -> y f16 [m, h]."""
        m, st = attn_out.shape[0], torch.cuda.current_stream().cuda_stream
        if m > self.q.shape[0]:
            raise ValueError(f"{m} tokens, workspaces hold {self.q.shape[0]}")
        s, sa = self.scales[0].data_ptr(), self.scales[1].data_ptr()
        api.norm_residual_q8(m, self.h, attn_out.data_ptr(), DT["f16"], self.q.data_ptr(), DT["i8"], s,
                             gain=self.gain.data_ptr(), post_gain=self.post_gain.data_ptr(),
                             residual=residual.data_ptr(), h=residual.data_ptr(), h_dtype=DT["bf16"], eps=EPS, stream=st)
        api.linear(m, self.f, self.h, DT["i8"], self.q.data_ptr(), self.gate[0].data_ptr(), self.a.data_ptr(), DT["f32"],
                   x_scale=s, w_scale=self.gate[1].data_ptr(), w_up=self.up[0].data_ptr(),
                   w_up_scale=self.up[1].data_ptr(), activation=api.ACTIVATIONS["gelu_tanh"], stream=st)
        api.quantize_rows(m, self.f, self.a.data_ptr(), DT["f32"], self.qa.data_ptr(), DT["i8"], sa, stream=st)
        api.linear(m, self.h, self.f, DT["i8"], self.qa.data_ptr(), self.down[0].data_ptr(), y.data_ptr(), DT["f16"],
                   x_scale=sa, w_scale=self.down[1].data_ptr(), stream=st)
        return y


def q8_0_rows(blocks, n, k):
    """n rows of k / 32 Q8_0 blocks as f32 on the device (exact)."""
    raw = torch.from_numpy(blocks.view(np.uint8).reshape(-1).copy()).cuda()
    out = torch.empty((n, k), device="cuda")
    api.q8_0_dequant(raw.data_ptr(), n * k // 32, out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    return out


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=4096)
    a = ap.parse_args(argv)
    rng = np.random.default_rng(0)
    hidden, ffn_len = synth.BASELINE.hidden, synth.BASELINE.ffn

    def weight(n, k):
        w = rng.standard_normal((n, k), dtype=np.float32) / np.float32(np.sqrt(k))
        return q8_0_rows(synth.quantize_q8_0(w), n, k)

    gate, up, down = weight(ffn_len, hidden), weight(ffn_len, hidden), weight(hidden, ffn_len)
    post, pre = (torch.from_numpy((1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32)).cuda() for _ in range(2))
    torch.manual_seed(0)
    m, h = a.tokens, gate.shape[1]
    attn = torch.randn((m, h), device="cuda").half()
    residual = (3 * torch.randn((m, h), device="cuda")).bfloat16()
    y = torch.empty((m, h), dtype=torch.float16, device="cuda")

    def rms(v):
        return v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS)

    want_h = residual.float() + rms(attn.float()) * post
    n = rms(want_h) * pre
    want = (torch.nn.functional.gelu(n @ gate.T, approximate="tanh") * (n @ up.T)) @ down.T

    ffn = Int8FeedForward(gate, up, down, post, pre, m)
    ffn(attn, residual, y)
    assert api.kernel_status(torch.cuda.current_device()) == 0
    err = float((y.float() - want).norm() / want.norm())
    cos = float(torch.nn.functional.cosine_similarity(y.float(), want).min())
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(20):
        ffn(attn, residual, y)
    end.record()
    end.synchronize()
    print(f"{m} tokens, {h} -> {gate.shape[0]} -> {h}: {start.elapsed_time(end) * 50:.1f} us a pass; against f32 "
          f"on the exact weights: relative error {err:.4f}, smallest row cosine {cos:.5f}")
    return err, cos


if __name__ == "__main__":
    main()
