"""What the source of the row operators' and the products' kernels promises, where no run can show that it is
kept."""
from __future__ import annotations

import os
import re

import pytest

from glypr_b200 import build


def code(name):
    """A source without its comments."""
    with open(os.path.join(build.CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


@pytest.mark.parametrize("name", ["linear_rows.cuh", "rowquant.cuh", "linear_any.cuh", "linear_tc.cuh", "linear_splitk.cuh"])
def test_dependent_launches_read_coherently(name):
    """A kernel that starts while the one before it still writes its operands may not read them through the
    non-coherent path, which asks for data that nothing writes during the kernel's life."""
    text = code(name)
    assert "griddep_wait" in text
    assert not re.search(r"__ldg\b|global\.nc\b|__ldlu\b|__ldcv\b", text)
