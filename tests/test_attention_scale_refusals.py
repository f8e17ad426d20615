"""Scales and caps whose quotient binary32 cannot hold are refused (no GPU needed)."""
import ctypes
import math

import pytest

from dgl_amd import _lib
from test_attention_refusals import step_struct, struct

BAD = [(0.25, 1e-40), (0.25, 1e-45), (1.0, 5e-39), (1e10, 1e-30), (-1e10, 1e-30), (math.inf, 1.0), (math.inf, 0.0), (2e38, 0.0),
       (0.25, math.nan)]
GOOD = [(0.25, 0.0), (0.0, 1e-30), (1e30, 1e-7), (-1e38, 0.0), (0.25, 2.0 ** -126), (0.25, 1e38)]


@pytest.mark.parametrize("scale,cap", BAD)
def test_refused(scale, cap):
    lib = _lib.load()
    a, b = struct(scale=scale, cap=cap), step_struct(scale=scale, cap=cap)
    assert lib.dgl_attention_forward(ctypes.byref(a), None, None) == -1 and b"scale" in lib.dgl_last_error_string()
    assert lib.dgl_attention_backward_workspace_floats(ctypes.byref(a)) == -1
    assert lib.dgl_attention_step(ctypes.byref(b), None, None) == -1 and b"scale" in lib.dgl_last_error_string()


@pytest.mark.parametrize("scale,cap", GOOD)
def test_taken(scale, cap):
    lib = _lib.load()
    assert lib.dgl_attention_backward_workspace_floats(ctypes.byref(struct(scale=scale, cap=cap))) > 0
    assert lib.dgl_attention_step_workspace_floats(ctypes.byref(step_struct(scale=scale, cap=cap))) >= 0


@pytest.mark.parametrize("cap", [1e-50, 1e-40, -1.0, math.nan, math.inf])
def test_python_refuses_a_cap_that_would_be_none(cap):
    from dgl_amd.attention import _cap
    with pytest.raises(ValueError, match="cap"):
        _cap(cap)
    assert _cap(0) == 0.0 and _cap(2.0 ** -126) == 2.0 ** -126
