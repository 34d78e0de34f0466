"""Gradient lists without a GPU: argument checks of the C ABI, and the layouts the
Python wrapper accepts.  No kernel is launched here."""
from __future__ import annotations

import ctypes

import pytest
import torch

from slmopt import GradientList, _lib
from slmopt.gradlist import _rows

BAD = _lib.SLM_ERR_INVALID_ARGUMENT


def view(data=4096, rows=1, columns=8, stride=8, dtype=_lib.DTYPE_F32):
    v = _lib.GradView()
    v.data, v.rows, v.columns, v.row_stride, v.dtype = data, rows, columns, stride, dtype
    return v


def create(*views, device=0):
    h = ctypes.c_void_p()
    arr = (_lib.GradView * max(1, len(views)))(*views)
    return _lib.load().slm_grad_list_create(arr, len(views), device, ctypes.byref(h)), h


def test_null_arguments_are_refused():
    lib = _lib.load()
    cfg = _lib.default_config()
    h = ctypes.c_void_p()
    one = ctypes.c_float(1.0)
    ptrs = (ctypes.c_void_p * 1)()
    calls = {
        "slm_grad_list_create": (None, 1, 0, ctypes.byref(h)),
        "slm_grad_list_bind": (None, ptrs, 1, None),
        "slm_grad_list_norm": (None, one, one, 0, None, None, None, None, None, 0, None),
        "slm_grad_list_clip": (None, None, one, one, 0, None, None, None, None, None, 0, None),
        "slm_grad_list_accumulate": (None, None, 0, 0, None),
        "slm_opt_step_list": (None, None, ctypes.byref(cfg), None, None),
        "slm_opt_norm_pass_list": (None, None, ctypes.byref(cfg), None),
        "slm_opt_norm_pass_accumulate_list": (None, None, None, 0, ctypes.byref(cfg), None),
    }
    for name, args in calls.items():
        assert getattr(lib, name)(*args) == BAD, name
        assert lib.slm_last_error_message().decode() != "no error", name
    assert lib.slm_grad_list_create((_lib.GradView * 1)(), 1, 0, None) == BAD
    assert lib.slm_grad_list_destroy(None) == _lib.SLM_OK
    assert lib.slm_grad_list_elements(None) == 0
    assert lib.slm_grad_list_workspace_bytes(None) == 0


@pytest.mark.parametrize("bad, status", [
    (dict(dtype=3), BAD),
    (dict(dtype=-1), BAD),
    (dict(rows=2, columns=8, stride=7), BAD),
    (dict(rows=2, columns=8, stride=0), BAD),
    (dict(rows=1 << 40, columns=1 << 40, stride=1 << 40), _lib.SLM_ERR_SIZE_LIMIT),
    (dict(rows=2, columns=8, stride=1 << 63), _lib.SLM_ERR_SIZE_LIMIT),
    (dict(rows=(1 << 64) - 1, columns=(1 << 64) - 1, stride=8), _lib.SLM_ERR_SIZE_LIMIT),
])
def test_bad_views_are_refused_before_any_device_is_touched(bad, status):
    got, h = create(view(), view(**bad))
    assert got == status and not h.value


def test_an_empty_list_is_refused():
    got, h = create()
    assert got == BAD and not h.value


def test_a_list_without_a_device_fails_cleanly():
    from conftest import have_gpu

    if have_gpu():
        pytest.skip("a GPU is visible")
    got, h = create(view())
    assert got == _lib.SLM_ERR_NO_DEVICE and not h.value


def test_list_total_beyond_any_memory_is_refused():
    big = view(rows=1, columns=1 << 47, stride=1 << 47)
    got, _ = create(big, big, big)
    assert got == _lib.SLM_ERR_SIZE_LIMIT


def test_layouts_the_wrapper_reads():
    x = torch.empty(6, 10)
    assert _rows(x) == (1, 60, 60)
    assert _rows(x[:, 2:7]) == (6, 5, 10)
    assert _rows(x[1:3]) == (1, 20, 20)
    assert _rows(x[::2]) == (3, 10, 20)
    assert _rows(x[:, 3]) == (6, 1, 10)
    assert _rows(x[:, :1]) == (6, 1, 10)
    assert _rows(torch.empty(0, 4)) == (1, 0, 0)
    assert _rows(torch.tensor(1.0)) == (1, 1, 1)
    y = torch.empty(4, 6, 10)
    assert _rows(y[:, :, :4]) == (24, 4, 10)          # rows at one distance across two dimensions
    assert _rows(y[:, :1, :]) == (4, 10, 60)
    assert _rows(y[:2].unsqueeze(1)) == (1, 120, 120)


@pytest.mark.parametrize("make", [
    lambda: torch.empty(6, 10).t(),
    lambda: torch.empty(1, 10).expand(6, 10),
    lambda: torch.empty(6, 10)[:, ::2][:, :3],
    lambda: torch.empty(4, 6, 10)[:, :3, :4],
    lambda: torch.empty(20).as_strided((4, 5), (3, 1)),
], ids=["transposed", "expanded", "every-other", "two-pitches", "overlapping"])
def test_layouts_the_wrapper_refuses(make):
    with pytest.raises(ValueError):
        _rows(make())


def test_the_wrapper_refuses_host_tensors_and_nothing():
    with pytest.raises(ValueError):
        GradientList([])
    with pytest.raises(ValueError):
        GradientList([torch.zeros(4)])
    with pytest.raises(ValueError):
        GradientList([[1.0, 2.0]])
