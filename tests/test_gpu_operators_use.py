"""glp_linear and the row operators as programs use them: residual in place on every kernel's path, from two
streams and two threads at once, without allocations, and erf-GELU held to its own error."""
from __future__ import annotations

import threading

import pytest

from glypr_b200 import api
from .test_gpu_operators import DT, Case, act64, buffer, filled, ptr, rows_of, run_quantize

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _lib():
    api.load_library()
    yield


@pytest.mark.parametrize("m,n,k,dtype,out,act,gated,pad,ypad", [
    (3, 520, 1000, "f16", "f16", "none", True, None, 0),          # few rows
    (20011, 520, 1000, "bf16", "bf16", "none", False, None, 0),   # CTA pairs, 8 and 16 epilogue warps, one to
    (20011, 520, 1000, "f16", "f32", "none", False, None, 0),     # four boxes of residual per warp
    (20011, 520, 1000, "bf16", "bf16", "gelu_erf", False, None, 0),
    (20011, 520, 1000, "f16", "f32", "gelu_erf", False, None, 0),
    (16385, 520, 2064, "i8", "f16", "silu", True, None, 0),
    (16385, 520, 2064, "e4m3", "f32", "gelu_tanh", True, None, 0),
    (20011, 777, 1000, "f16", "f16", "relu", False, None, 0),     # rows off 16 bytes: column by column
    (16385, 520, 1056, "bf16", "f32", "silu", True, None, 3),
    (700, 520, 192, "f16", "bf16", "none", False, None, 0),       # single CTAs
    (700, 521, 192, "i8", "f32", "none", True, None, 0),
    (100, 300, 3000, "f16", "f16", "none", False, None, 0),       # K split over a cluster
    (128, 64, 8100, "i8", "f32", "silu", True, None, 3),
    (40, 203, 176, "f16", "f16", "gelu_tanh", False, 1, 0),       # operands off 16-byte rows
    (300, 203, 176, "e4m3", "bf16", "silu", True, 5, 1),
])
def test_residual_in_place(m, n, k, dtype, out, act, gated, pad, ypad):
    """y = residual gives the bits that an output of its own gives, in every row."""
    c = Case(m, n, k, dtype, out, act=act, gated=gated, bias=True, res=True, seed=m + n, pad=pad, ypad=ypad)
    apart = c.run().clone()
    c.check(slice(-70, None))
    c.run(y=c.res)
    assert torch.equal(c.res, apart)


def mixed_cases(seed):
    """A product for each kernel, and their outputs one after the other."""
    sizes = [(2, 768, 768, "f16"), (12, 2400, 1152, "i8"), (100, 300, 3000, "e4m3"), (513, 768, 768, "bf16"),
             (9000, 768, 1152, "f16"), (9000, 300, 768, "i8"), (33, 130, 100, "f16")]
    cases = [Case(m, n, k, d, "f32", act="gelu_tanh", gated=i % 2 == 1, bias=True, res=True, seed=seed + i,
                  pad=1 if m == 33 else None) for i, (m, n, k, d) in enumerate(sizes)]
    alone = []
    for c in cases:
        alone.append(c.run().clone())
        torch.cuda.synchronize()
        c.y.fill_(float("nan"))
    torch.cuda.synchronize()
    return cases, alone


def test_two_streams_at_once():
    sets = [mixed_cases(100), mixed_cases(200)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for i in range(len(sets[0][0])):
            for (cases, _), st in zip(sets, streams):
                cases[i].run(stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert api.kernel_status(torch.cuda.current_device()) == 0
    for cases, alone in sets:
        for c, y in zip(cases, alone):
            assert torch.equal(c.y, y)


def test_two_threads_at_once():
    sets = [mixed_cases(300), mixed_cases(400)]
    failed = []

    def work(cases):
        try:
            st = torch.cuda.Stream()
            for _ in range(20):
                for c in cases:
                    c.run(stream=st.cuda_stream)
            st.synchronize()
            with pytest.raises(api.GlyprError) as e:  # messages are the thread's own
                api.linear(4, 0, 8, DT["f16"], 16, 16, 16, DT["f16"])
            assert "N >= 1" in e.value.message
        except BaseException as e:
            failed.append(e)
    threads = [threading.Thread(target=work, args=(cases,)) for cases, _ in sets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    torch.cuda.synchronize()
    for cases, alone in sets:
        for c, y in zip(cases, alone):
            assert torch.equal(c.y, y)


def test_nothing_is_allocated_after_the_first_call():
    cases, _ = mixed_cases(500)
    x, q, s = filled(rows_of(500, 1152, 1), "f16"), buffer(500, 1152, "i8"), torch.empty(500, device="cuda")

    def everything():
        for c in cases:
            c.run()
        run_quantize(x, q, s, "f16", "i8")
        api.norm_residual_q8(500, 1152, ptr(x), DT["f16"], ptr(q), DT["i8"], ptr(s), residual=ptr(x), h_dtype=DT["f16"])
        torch.cuda.synchronize()
    everything()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(3):
        everything()
    assert torch.cuda.mem_get_info()[0] == free


@pytest.mark.parametrize("m", [1, 64, 300])
def test_erf_gelu_to_its_error(m):
    """0.5 |v| erfc(|v| / sqrt 2) is 2 to an exponent of E = 0.72 v^2 and less: its product, its constant and its sum
    are each rounded by up to 2^-24 of E; beside that the fit's 9e-7 and some ulps of f32."""
    v = torch.linspace(-14, 14, 3001, device="cuda").half()
    c = Case(m, v.numel(), 1, "f16", "f32", act="gelu_erf", seed=1)
    c.w[:, 0] = v
    c.x[:, 0] = 1.0
    c.run()
    v = v.double()
    want = act64(v, "gelu_erf")
    bound = (2e-6 + 3 * 0.6931 * 2.0 ** -24 * 0.7213475 * v * v) * want.abs() + 1.2e-37
    assert ((c.y.double() - want).abs() <= bound).all()
    near = v.abs() <= 1
    assert ((c.y.double() - want).abs() <= 1.5e-6 * want.abs())[:, near].all()
