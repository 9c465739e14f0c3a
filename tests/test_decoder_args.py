"""Argument checks of the decoder operators that need no GPU: the C entries report errors before they launch
anything, the Python entries refuse tensors that are not on a GPU."""
import ctypes as C

import pytest
import torch

from d3gs_research_b200 import _lib, group_norm_act


def gn_desc(**kw):
    d = _lib.GroupNorm()
    for k, v in dict(batch=1, pixels=4, channels=8, groups=2, x_batch_stride=32, x_pixel_stride=8, dy_batch_stride=32,
                     dy_pixel_stride=8, dtype=0, weight_dtype=0, act=1, eps=1e-5, **kw).items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("field,value,word", [("groups", 3, "divide"), ("groups", 0, "divide"), ("channels", 0, "channels"),
                                              ("channels", 16385, "channels"), ("batch", 65536, "batch"), ("batch", -1, "batch"),
                                              ("dtype", 3, "dtype"), ("weight_dtype", -1, "dtype"), ("act", 3, "act"),
                                              ("eps", -1.0, "eps"), ("eps", float("nan"), "eps")])
def test_group_norm_descriptor(field, value, word):
    lib = _lib.load()
    d = gn_desc()
    setattr(d, field, value)
    assert lib.d3gs_group_norm_workspace_bytes(C.byref(d), 0) == 0
    assert word in _lib.last_error()
    assert lib.d3gs_group_norm_forward(C.byref(d), 16, None, None, 16, 16, 16, 1 << 20, None) == -1
    assert lib.d3gs_group_norm_backward(C.byref(d), 16, None, None, 16, 16, 16, None, None, 16, 1 << 20, None) == -1


def test_group_norm_pointers_and_workspace():
    lib = _lib.load()
    d = gn_desc()
    need = lib.d3gs_group_norm_workspace_bytes(C.byref(d), 0)
    assert need > 0
    assert lib.d3gs_group_norm_forward(None, 16, None, None, 16, 16, 16, need, None) == -1
    assert lib.d3gs_group_norm_forward(C.byref(d), None, None, None, 16, 16, 16, need, None) == -1
    assert lib.d3gs_group_norm_forward(C.byref(d), 16, None, None, 16, 16, 16, need - 1, None) == -1
    assert "workspace" in _lib.last_error()
    assert lib.d3gs_group_norm_forward(C.byref(d), 16, None, None, 16, 16, 24, need, None) == -1
    assert lib.d3gs_group_norm_backward(C.byref(d), 16, None, None, 16, 16, None, None, None, 16, 1 << 20, None) == -1
    assert "no gradient" in _lib.last_error()
    for field in ("batch", "pixels"):           # nothing to do: nothing is launched, nothing is read
        e = gn_desc()
        setattr(e, field, 0)
        assert lib.d3gs_group_norm_workspace_bytes(C.byref(e), 0) > 0
        assert lib.d3gs_group_norm_workspace_bytes(C.byref(e), 1) > 0
        assert lib.d3gs_group_norm_forward(C.byref(e), None, None, None, None, None, None, 0, None) == 0


def test_group_norm_needs_a_gpu_tensor():
    with pytest.raises(ValueError, match="CUDA tensor"):
        group_norm_act(torch.zeros(1, 2, 2, 8), 2)
