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
                                              ("x_pixel_stride", -8, "strides"), ("dy_batch_stride", -1, "strides"),
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


def ortho(count=1, **kw):
    mats = (_lib.OrthoMatrix * count)()
    for m in mats:
        m.src, m.dst, m.momentum, m.rows, m.cols, m.src_row_stride, m.rate = 16, 16, 16, 4, 6, 6, 0.1
        for k, v in kw.items():
            setattr(m, k, v)
    cfg = _lib.OrthoConfig()
    cfg.steps, cfg.eps = 5, 1e-7
    for k in range(5):
        cfg.coefficients[k][:] = (3.4445, -4.775, 2.0315)
    return mats, cfg


@pytest.mark.parametrize("kw,word", [({"rows": 16385, "cols": 16385}, "short side"), ({"cols": 1 << 25}, "long side"),
                                     ({"rows": -1}, "short side"), ({"src": None}, "NULL"), ({"dst": None}, "NULL"),
                                     ({"src_row_stride": -1}, "stride")])
def test_ortho_matrix(kw, word):
    lib = _lib.load()
    mats, cfg = ortho(**kw)
    assert lib.d3gs_orthogonalize(mats, 1, C.byref(cfg), 256, 1 << 40, None) == -1
    assert word in _lib.last_error()
    assert lib.d3gs_muon_step(mats, 1, C.byref(cfg), 256, 1 << 40, None) == -1


@pytest.mark.parametrize("kw,word", [({"steps": 0}, "steps"), ({"steps": 33}, "steps"), ({"eps": 0.0}, "eps"),
                                     ({"eps": float("nan")}, "eps"), ({"dtype": 2}, "dtype")])
def test_ortho_config(kw, word):
    lib = _lib.load()
    mats, cfg = ortho()
    for k, v in kw.items():
        setattr(cfg, k, v)
    assert lib.d3gs_orthogonalize_workspace_bytes(mats, 1, C.byref(cfg)) == 0
    assert lib.d3gs_orthogonalize(mats, 1, C.byref(cfg), 256, 1 << 40, None) == -1
    assert word in _lib.last_error()


def test_ortho_coefficients_that_grow_without_bound():
    lib = _lib.load()
    mats, cfg = ortho()
    for k in range(5):
        cfg.coefficients[k][:] = (5.0, 0.0, 0.0)          # 5^5 = 3125
    assert lib.d3gs_orthogonalize(mats, 1, C.byref(cfg), 256, 1 << 40, None) == -1
    assert "singular values grow" in _lib.last_error()
    for k in range(5):
        cfg.coefficients[k][:] = (1.5, -0.5, 1e-4)
    assert lib.d3gs_orthogonalize(mats, 1, C.byref(cfg), 256, 1 << 40, None) == -1
    assert "b / c" in _lib.last_error()
    for k in range(5):
        cfg.coefficients[k][:] = (0.0, 0.0, 0.0)
    assert lib.d3gs_orthogonalize_workspace_bytes(mats, 1, C.byref(cfg)) > 0


def test_ortho_workspace():
    lib = _lib.load()
    mats, cfg = ortho(3)
    need = lib.d3gs_orthogonalize_workspace_bytes(mats, 3, C.byref(cfg))
    assert need >= lib.d3gs_orthogonalize_workspace_bytes(mats, 1, C.byref(cfg)) > 0
    for ws, n in ((None, need), (256, need - 1), (264, need)):
        assert lib.d3gs_orthogonalize(mats, 3, C.byref(cfg), ws, n, None) == -1
        assert "workspace" in _lib.last_error()
    assert lib.d3gs_orthogonalize(None, 2, C.byref(cfg), 256, need, None) == -1
    assert lib.d3gs_orthogonalize(mats, 3, None, 256, need, None) == -1
    mats[0].momentum = None
    assert lib.d3gs_muon_step(mats, 3, C.byref(cfg), 256, need, None) == -1
    cfg.dtype = 1
    assert lib.d3gs_muon_step(mats, 3, C.byref(cfg), 256, need, None) == -1
    # no matrices, or only empty ones: nothing is launched
    cfg.dtype = 0
    assert lib.d3gs_orthogonalize(None, 0, C.byref(cfg), 256, 256, None) == 0
    mats, cfg = ortho(2, rows=0, src=None, dst=None)
    assert lib.d3gs_orthogonalize(mats, 2, C.byref(cfg), 256, 1 << 20, None) == 0


def test_coefficients_are_taken_by_value():
    from d3gs_research_b200 import muon
    a = torch.tensor(1.5)
    first = muon._config("x", 0, (a, -0.5, 0.0), 1e-7, 2)
    a.fill_(2.0)
    second = muon._config("x", 0, [[a, -0.5, 0.0]] * 2, 1e-7, 2)
    assert first.coefficients[0][0] == first.coefficients[1][0] == 1.5
    assert second.coefficients[0][0] == second.coefficients[1][0] == 2.0
    assert first.coefficients[0][1] == -0.5 and first.steps == 2


def test_muon_needs_gpu_tensors():
    from d3gs_research_b200 import GaussianMuon, muon_step, orthogonalize
    u = torch.zeros(4, 6)
    with pytest.raises(ValueError, match="CUDA tensor"):
        orthogonalize(u)
    with pytest.raises(ValueError, match="CUDA tensors"):
        muon_step([u], [u.clone()], [u.clone()], lr=0.1)
    for kw in ({"ns_steps": 0}, {"eps": -1.0}, {"ns_coefficients": (1.0,)}):
        with pytest.raises(ValueError, match="GaussianMuon"):
            GaussianMuon([torch.nn.Parameter(u)], **kw)
    with pytest.raises(ValueError, match="two or more axes"):
        GaussianMuon([torch.nn.Parameter(torch.zeros(4))])
