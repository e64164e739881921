"""Sizes beyond the C interface's integers: refused as every other argument is, not taken modulo 2^32."""
from __future__ import annotations

import pytest

from glypr_b200 import api

DT = api.DTYPES
P = 1 << 20  # a stand-in address, never touched


@pytest.mark.parametrize("size", [2 ** 31, 2 ** 32, 2 ** 32 + 4, -2 ** 31 - 1, 2 ** 70])
@pytest.mark.parametrize("call", [
    lambda v: api.quantize_rows(v, 16, P, DT["f16"], P, DT["i8"], P),
    lambda v: api.quantize_rows(4, v, P, DT["f16"], P, DT["i8"], P),
    lambda v: api.norm_residual_q8(v, 16, P, DT["f16"], P, DT["i8"], P),
    lambda v: api.norm_residual_q8(4, v, P, DT["f16"], P, DT["i8"], P),
    lambda v: api.linear(v, 8, 16, DT["f16"], P, P, P, DT["f16"]),
    lambda v: api.linear(4, v, 16, DT["f16"], P, P, P, DT["f16"]),
    lambda v: api.linear(4, 8, v, DT["f16"], P, P, P, DT["f16"]),
    lambda v: api.linear(4, 8, 16, v, P, P, P, DT["f16"]),
])
def test_sizes_beyond_an_int(call, size):
    with pytest.raises(api.GlyprError) as e:
        call(size)
    assert e.value.code == api.GLP_ERR_INVALID_ARG
