"""What the operators around the step refuse, before anything is launched: no GPU is needed."""

import ctypes

import numpy as np
import pytest
import torch

import apexw_amd
from apexw_amd import _lib


def test_layer_norm_refuses():
    x, w = torch.randn(4, 8), torch.ones(8)
    with pytest.raises(ValueError, match="GPU"):
        apexw_amd.layer_norm_forward(x, w, w)
    with pytest.raises(TypeError, match="float64"):
        apexw_amd.layer_norm_forward(x.double())
    with pytest.raises(ValueError, match="at least one element"):
        apexw_amd.layer_norm_forward(torch.randn(4, 0))
    with pytest.raises(ValueError, match="at least one element"):
        apexw_amd.layer_norm_forward(torch.tensor(1.0))


def test_expert_matmul_refuses():
    x, w = torch.randn(4, 8).bfloat16(), torch.randn(2, 6, 8).bfloat16()
    ends = torch.tensor([1, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        apexw_amd.expert_matmul_forward(x, w, ends)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        apexw_amd.expert_matmul_forward(x.float(), w.float(), ends)
    with pytest.raises(ValueError, match="rows"):
        apexw_amd.expert_matmul_weight_grad(x[0], x, ends)


def test_clip_refuses():
    g = [torch.randn(4)]
    with pytest.raises(ValueError, match="GPU"):
        apexw_amd.clip_grads(g, 1.0)
    with pytest.raises(ValueError, match="norm_type"):
        apexw_amd.clip_grads(g, 1.0, 3.0)
    with pytest.raises(ValueError, match="max_norm"):
        apexw_amd.clip_grads(g, -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        apexw_amd.clip_grads(g, float("nan"))
    with pytest.raises(ValueError, match="copies"):
        apexw_amd.clip_grads(g, 1.0, out=[])
    with pytest.raises(TypeError, match="tensors"):
        apexw_amd.clip_grads([1.0], 1.0)
    assert float(apexw_amd.clip_grads([], 1.0)) == 0.0


def test_entry_points_refuse_without_launching():
    lib, ok = _lib.load(), 4096        # an aligned address that no call here reaches
    fwd, bwd = lib.apexw_layer_norm_forward, lib.apexw_layer_norm_backward
    F32, BF16, F16 = _lib.F32, _lib.BF16, _lib.F16
    assert fwd(None, 1, 8, 8, F32, ok, ok, F32, 1e-5, ok, ok, ok, None) == 1
    assert fwd(ok, -1, 8, 8, F32, ok, ok, F32, 1e-5, ok, ok, ok, None) == 1
    assert fwd(ok, 1, 0, 8, F32, ok, ok, F32, 1e-5, ok, ok, ok, None) == 1
    assert fwd(ok, 1, 8, -8, F32, ok, ok, F32, 1e-5, ok, ok, ok, None) == 1
    assert fwd(ok, 1, 8, 8, F32, ok, ok, F32, float("nan"), ok, ok, ok, None) == 1
    assert fwd(ok, 1, 8, 8, F32, ok, ok, BF16, 1e-5, ok, ok, ok, None) == 2
    assert fwd(ok, 1, 8, 8, BF16, ok, ok, F16, 1e-5, ok, ok, ok, None) == 2
    assert fwd(ok, 1, 8, 8, 7, ok, ok, F32, 1e-5, ok, ok, ok, None) == 2
    assert fwd(ok + 2, 1, 8, 8, F32, ok, ok, F32, 1e-5, ok, ok, ok, None) == 4
    assert fwd(ok + 1, 1, 8, 8, BF16, ok, ok, F32, 1e-5, ok, ok, ok, None) == 4
    assert bwd(ok, 8, ok, 8, ok, ok, ok, 1, 8, F32, F32, ok, ok, ok, None, None) == 1     # no workspace
    assert bwd(ok, 8, ok, 8, None, ok, ok, 1, 8, F32, F32, ok, ok, ok, ok, None) == 1
    assert bwd(ok, 8, ok, 8, ok, ok, ok, 1, 8, F16, BF16, ok, ok, ok, ok, None) == 2
    assert bwd(ok, 8, ok, 8, ok, ok, ok, 1, 8, F32, F32, ok, ok + 1, ok, ok, None) == 4
    assert lib.apexw_layer_norm_workspace(-1, 8) == -1 and lib.apexw_layer_norm_workspace(5, 0) == -1
    assert lib.apexw_layer_norm_workspace(5, 8) >= 80

    rows, grad = lib.apexw_expert_rows, lib.apexw_expert_weight_grad
    assert rows(None, 8, ok, 8, 64, 0, ok, 2, 4, 8, 8, BF16, ok, 8, None, None) == 1
    assert rows(ok, 8, ok, 8, 64, 2, ok, 2, 4, 8, 8, BF16, ok, 8, None, None) == 1
    assert rows(ok, 8, ok, 8, 64, 0, ok, 0, 4, 8, 8, BF16, ok, 8, None, None) == 1
    assert rows(ok, 8, ok, 8, 64, 0, ok, 2, 4, 0, 8, BF16, ok, 8, None, None) == 1
    assert rows(ok, 8, ok, 8, 64, 0, ok, 2, 4, 8, 8, BF16, ok, 7, None, None) == 1
    assert rows(ok, 8, ok, 8, 64, 0, ok, 2, 4, 8, 8, F32, ok, 8, None, None) == 2
    assert rows(ok + 1, 8, ok, 8, 64, 0, ok, 2, 4, 8, 8, BF16, ok, 8, None, None) == 4
    assert rows(ok, 8, ok, 8, 64, 0, ok + 2, 2, 4, 8, 8, BF16, ok, 8, None, None) == 4
    assert rows(ok, 8, ok, 8, 64, 0, ok, 2, 2 ** 31 - 1, 8, 2 ** 31 - 300, BF16, ok, 2 ** 31, None, None) == 5
    assert grad(ok, 8, ok, 8, ok, 2, 4, 8, 8, BF16, ok, F16, None, None) == 2
    assert grad(ok, 8, ok, 8, ok, 2, 4, 8, 8, F32, ok, F32, None, None) == 2
    assert grad(ok, 8, ok, 8, ok, 2, 4, 8, 8, BF16, ok + 2, F32, None, None) == 4
    assert grad(None, 8, ok, 8, ok, 2, 4, 8, 8, BF16, ok, F32, None, None) == 1
    assert grad(ok, 8, ok, 8, ok, 2 ** 20, 4, 2 ** 20, 2 ** 20, BF16, ok, F32, None, None) == 5

    norm, scale, clip = lib.apexw_grad_norm, lib.apexw_grad_scale, lib.apexw_clip_grads
    assert norm(ok, 1, 1, 3, ok, ok, None) == 1 and norm(ok, 1, 1, 2, None, ok, None) == 1
    assert norm(None, 1, 1, 2, ok, ok, None) == 1 and norm(ok, 0, 1, 2, ok, ok, None) == 1
    assert scale(ok, 1, 1, None, 1.0, None) == 1 and scale(ok, 1, 1, ok, -1.0, None) == 1
    assert scale(ok, 1, 1, ok, float("nan"), None) == 1 and scale(None, 0, 0, ok, 1.0, None) == 0
    assert clip(ok, 1, 1, 2, -1.0, ok, ok, None) == 1 and clip(ok, 1, -1, 2, 1.0, ok, ok, None) == 1


def test_clip_layout():
    t = np.zeros(4, dtype=_lib.CLIP_TENSOR_DTYPE)
    t["g"], t["out"], t["n"] = 4096, 8192, [8192, 0, 8193, 1]
    lay = _lib.load().apexw_clip_layout
    assert lay(t.ctypes.data, 4) == 4 and t["first_unit"].tolist() == [0, 1, 1, 3]
    assert lay(t.ctypes.data, 0) == 0 and lay(None, 1) == -1
    for field, value, status in (("n", -1, -1), ("g", 0, -1), ("g", 4098, -4), ("out", 8193, -4), ("g_dtype", 3, -2),
                                 ("out_dtype", 4, -2)):
        bad = t.copy()
        bad[field][2] = value
        assert lay(bad.ctypes.data, 4) == status, field
    assert ctypes.sizeof(ctypes.c_void_p) == 8
