"""Errors of the row operators and glp_linear that the CUDA runtime finds, not their own checks."""
from __future__ import annotations

import ctypes

import pytest

from glypr_b200 import api

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = api.DTYPES


def calls():
    x = torch.ones((4, 64), dtype=torch.float16, device="cuda")
    q, s = torch.empty((4, 64), dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    y = torch.empty((4, 4), dtype=torch.float16, device="cuda")
    return {
        "quantize": lambda: api.quantize_rows(4, 64, x.data_ptr(), DT["f16"], q.data_ptr(), DT["i8"], s.data_ptr()),
        "norm": lambda: api.norm_residual_q8(4, 64, x.data_ptr(), DT["f16"], q.data_ptr(), DT["i8"], s.data_ptr()),
        "linear": lambda: api.linear(4, 4, 64, DT["f16"], x.data_ptr(), x.data_ptr(), y.data_ptr(), DT["f16"]),
    }


@pytest.mark.parametrize("name", ["quantize", "norm", "linear"])
def test_a_refused_launch_is_reported_once(name):
    """A launch on the default stream is refused while another stream is being captured.  The call says so; the
    next call of the library, after the capture, does not."""
    api.load_library()
    call = calls()[name]
    blocks = torch.zeros(34, dtype=torch.uint8, device="cuda")
    out = torch.full((32,), float("nan"), device="cuda")
    call()
    torch.cuda.synchronize()
    cu = ctypes.CDLL("libcuda.so.1")
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert cu.cuStreamCreate(ctypes.byref(stream), 0) == 0
    try:
        assert cu.cuStreamBeginCapture_v2(stream, 2) == 0  # relaxed; refused all the same: the two are ordered
        try:
            with pytest.raises(api.GlyprError) as e:
                call()
        finally:
            cu.cuStreamEndCapture(stream, ctypes.byref(graph))
        assert e.value.code == api.GLP_ERR_CUDA and "launch" in e.value.message
        api.q8_0_dequant(blocks.data_ptr(), 1, out.data_ptr())
        call()
        torch.cuda.synchronize()
        assert (out == 0).all()
    finally:
        if graph:
            cu.cuGraphDestroy(graph)
        cu.cuStreamDestroy_v2(stream)
