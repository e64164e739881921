"""The row operators and glp_linear in rows of calls that write and read the same buffers: each call sees
what the calls before it in the stream wrote, though it may start while they still run."""
from __future__ import annotations

import pytest

from glypr_b200 import api

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = api.DTYPES
ROUNDS = 150


@pytest.fixture(scope="module", autouse=True)
def _lib():
    api.load_library()
    yield


def randn(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream


def eager_and_graph(step, outputs):
    """step(i) for i in range(ROUNDS): one call at a time, then in a row, then from a graph; the values that
    each way leaves in `outputs` have to be the same."""
    got = []
    for way in ("alone", "row", "graph"):
        outputs.fill_(float("nan"))
        torch.cuda.synchronize()
        if way == "graph":
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                for i in range(ROUNDS):
                    step(i, lambda: None)
            outputs.fill_(float("nan"))
            g.replay()
        else:
            for i in range(ROUNDS):
                step(i, torch.cuda.synchronize if way == "alone" else lambda: None)
        torch.cuda.synchronize()
        got.append(outputs.clone())
    assert not got[0].isnan().any()
    assert torch.equal(got[1], got[0]) and torch.equal(got[2], got[0])


@pytest.mark.parametrize("m", [1, 7, 16, 30])
@pytest.mark.parametrize("dtype", ["i8", "e4m3"])
def test_few_rows_product_of_rows_just_quantised(m, dtype):
    """Rows quantised into one buffer, multiplied, quantised anew, ...: new values each time."""
    n, k = 768, 1152
    x = randn(m, ROUNDS, m, k).half()
    w8 = torch.empty((n, k), dtype=torch.int8, device="cuda")
    ws = torch.empty(n, device="cuda")
    w = randn(1, n, k)
    api.quantize_rows(n, k, w.data_ptr(), DT["f32"], w8.data_ptr(), DT[dtype], ws.data_ptr(), stream=stream())
    q, s = torch.empty((m, k), dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    y = torch.empty((ROUNDS, m, n), device="cuda")

    def step(i, between):
        api.quantize_rows(m, k, x[i].data_ptr(), DT["f16"], q.data_ptr(), DT[dtype], s.data_ptr(), stream=stream())
        between()
        api.linear(m, n, k, DT[dtype], q.data_ptr(), w8.data_ptr(), y[i].data_ptr(), DT["f32"], x_scale=s.data_ptr(),
                   w_scale=ws.data_ptr(), stream=stream())
        between()
    eager_and_graph(step, y)
    want = x.double() @ w.double().T
    assert float((y.double() - want).norm() / want.norm()) < 0.06  # 8-bit rows: at most 2^-4 of a value's binade each


@pytest.mark.parametrize("gated", [False, True])
def test_few_rows_product_of_weights_just_quantised(gated):
    """The weights' codes and scales rewritten before each product."""
    m, n, k = 3, 400, 768
    w = randn(5, ROUNDS, n, k).bfloat16()
    x8, xs = torch.empty((m, k), dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    x = randn(6, m, k)
    api.quantize_rows(m, k, x.data_ptr(), DT["f32"], x8.data_ptr(), DT["i8"], xs.data_ptr(), stream=stream())
    q, s = torch.empty((n, k), dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    up = dict(w_up=q.data_ptr(), w_up_scale=s.data_ptr()) if gated else {}
    y = torch.empty((ROUNDS, m, n), device="cuda")

    def step(i, between):
        api.quantize_rows(n, k, w[i].data_ptr(), DT["bf16"], q.data_ptr(), DT["i8"], s.data_ptr(), stream=stream())
        between()
        api.linear(m, n, k, DT["i8"], x8.data_ptr(), q.data_ptr(), y[i].data_ptr(), DT["f32"], x_scale=xs.data_ptr(),
                   w_scale=s.data_ptr(), stream=stream(), **up)
        between()
    eager_and_graph(step, y)


@pytest.mark.parametrize("m", [2, 12, 40])
def test_products_in_a_chain(m):
    """Each product's x is the last one's y, over two buffers."""
    k = 512
    w = (randn(7, k, k) / k ** 0.5).half()
    bufs = [randn(8, m, k).half(), torch.empty((m, k), dtype=torch.float16, device="cuda")]
    first = bufs[0].clone()

    def step(i, between):
        if i == 0:
            bufs[0].copy_(first)
        api.linear(m, k, k, DT["f16"], bufs[i % 2].data_ptr(), w.data_ptr(), bufs[1 - i % 2].data_ptr(), DT["f16"],
                   activation=api.ACTIVATIONS["gelu_tanh"], residual=first.data_ptr(), stream=stream())
        between()
    assert ROUNDS % 2 == 0
    eager_and_graph(step, bufs[0])


@pytest.mark.parametrize("h", [64, 768, 771, 1152, 2051, 9000])
def test_norm_with_gains_just_written(h):
    """Both gains are rows that the product before the norm wrote, new ones each time."""
    m, k = 40, 16
    src = randn(h, ROUNDS, 2, k).half()
    w = (randn(h + 1, h, k) / 4).half()
    x, res = randn(h + 2, m, h).half(), randn(h + 3, m, h).bfloat16()
    pitch = (h + 3) // 4 * 4
    gains = torch.empty((2, pitch), device="cuda")
    q, s = torch.empty((ROUNDS, m, h), dtype=torch.int8, device="cuda"), torch.empty((ROUNDS, m), device="cuda")
    hout = torch.empty((m, h), dtype=torch.bfloat16, device="cuda")
    outs = torch.empty((ROUNDS, m, h + 1), device="cuda")

    def step(i, between):
        api.linear(2, h, k, DT["f16"], src[i].data_ptr(), w.data_ptr(), gains.data_ptr(), DT["f32"], ldy=pitch, stream=stream())
        between()
        api.norm_residual_q8(m, h, x.data_ptr(), DT["f16"], q[i].data_ptr(), DT["i8"], s[i].data_ptr(),
                             gain=gains[0].data_ptr(), post_gain=gains[1].data_ptr(), residual=res.data_ptr(),
                             h=hout.data_ptr(), h_dtype=DT["bf16"], stream=stream())
        between()
        if i == ROUNDS - 1:
            outs[:, :, :h].copy_(q)
            outs[:, :, h].copy_(s)
    eager_and_graph(step, outs)
    # the last round's rows against the formula; int8 codes: half a step of 1 / 127 of the row's largest value
    post, gain = ((src[-1, r].double() @ w.double().T) for r in (1, 0))

    def rms(v):
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6)
    n = rms(res.double() + rms(x.double()) * post) * gain
    err = (q[-1].double() * s[-1].double()[:, None] - n).abs()
    assert (err <= 0.501 * n.abs().amax(1, keepdim=True) / 127).all()
