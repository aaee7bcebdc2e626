"""Refusals of the operators on rows of logits and on gradients, in Python and at the C ABI: every one
of them is decided on the host, before anything reaches a GPU."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from bayesiannetwork_amd.inference_machines.hip_spa import _native
from bayesiannetwork_amd.optimizers import (
    HipGradientClipper,
    states_log_likelihood,
    states_log_likelihood_and_gradient,
)
from bayesiannetwork_amd.samplers import draw_states

LOGITS, U, STATES = torch.zeros((3, 4)), torch.zeros(3), torch.zeros(3, dtype=torch.int64)


@pytest.mark.parametrize("call", [
    lambda x: draw_states(x, U),
    lambda x: states_log_likelihood(x, STATES),
    lambda x: states_log_likelihood_and_gradient(x, STATES),
], ids=["draw", "likelihood", "gradient"])
@pytest.mark.parametrize("logits,error,match", [
    (LOGITS, ValueError, "no CPU path"),
    (LOGITS.long(), TypeError, "float32"),
    (LOGITS[0], ValueError, "rows, states"),
    (torch.zeros((3, 0)), ValueError, "at least one state"),
    ([[0.0]], TypeError, "tensor"),
])
def test_logits_are_checked(call, logits, error, match):
    with pytest.raises(error, match=match):
        call(logits)


@pytest.mark.parametrize("gradients,error,match", [
    ([], ValueError, "no gradients"),
    ([torch.zeros(3)], ValueError, "no CPU path"),
    ([torch.zeros(3, dtype=torch.int32)], TypeError, "float32"),
    ([3.0], TypeError, "tensor"),
])
def test_gradients_are_checked(gradients, error, match):
    with pytest.raises(error, match=match):
        HipGradientClipper(gradients)


# addresses that are never read: the checks come first
A, B = 1 << 20, 1 << 24


def _draw(dtype=0, logits=A, rows=3, states=4, stride=4, counts=None, u_dtype=0, u=B, workspace=B, out=B, **filters):
    f = _native.DrawFilters(1.0, 0, 1.0, 0.0)
    for k, v in filters.items():
        setattr(f, k, v)
    return _native.load().bn_draw_states(dtype, logits, rows, states, stride, counts, u_dtype, u, ctypes.byref(f),
                                         workspace, out, None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=4), "dtype"), (dict(dtype=-1), "dtype"), (dict(rows=-1), "rows"), (dict(states=0), "num_states"),
    (dict(states=(1 << 24) + 1), "num_states"), (dict(stride=-4), "stride"), (dict(u_dtype=2), "uniform_dtype"),
    (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(top_k=-1), "top_k"), (dict(top_p=0.0), "top_p"),
    (dict(top_p=1.5), "top_p"), (dict(top_p=float("nan")), "top_p"), (dict(min_p=-0.1), "min_p"),
    (dict(min_p=1.1), "min_p"), (dict(logits=None), "null"), (dict(u=None), "null"), (dict(out=None), "null"),
    (dict(workspace=None, states=2049), "null"), (dict(workspace=B + 4, states=2049), "aligned"),
    (dict(logits=A + 2), "aligned"),
])
def test_draw_refusals(change, message):
    assert _draw(**change) == -1
    assert message in _native.load().bn_last_error().decode()


def test_draw_of_no_rows_and_workspace_sizes():
    lib = _native.load()
    assert _draw(rows=0, logits=None, u=None, out=None, workspace=None) == 0
    assert lib.bn_draw_states_workspace_bytes(0, 3, 2048) == 0
    assert lib.bn_draw_states_workspace_bytes(0, 3, 2049) > 0
    for bad in ((7, 3, 4), (0, -1, 4), (0, 3, 0), (0, 3, (1 << 24) + 1)):
        assert lib.bn_draw_states_workspace_bytes(*bad) == -1


def _gradient(dtype=0, logits=A, rows=3, states=4, stride=4, s=B, state_bytes=8, totals=None, weights=None, w_stride=0,
              ll=None, gradient=B, g_stride=4):
    return _native.load().bn_states_log_likelihood_gradient(dtype, logits, rows, states, stride, None, s, state_bytes,
                                                            totals, weights, w_stride, ll, gradient, g_stride, None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=9), "dtype"), (dict(rows=-1), "rows"), (dict(states=0), "num_states"), (dict(state_bytes=2), "1, 4 or 8"),
    (dict(logits=None), "null"), (dict(s=None), "null"), (dict(gradient=None), "null"), (dict(g_stride=3), "overlap"),
    (dict(stride=-1), "stride"), (dict(weights=B, w_stride=-1), "stride"), (dict(totals=B, ll=B), "either"),
    (dict(gradient=A + 4), "lies over"), (dict(gradient=A, g_stride=5), "lies over"), (dict(logits=A + 1), "aligned"),
    (dict(gradient=B + 2), "aligned"), (dict(gradient=A, stride=0), "lies over"),
])
def test_likelihood_refusals(change, message):
    assert _gradient(**change) == -1
    assert message in _native.load().bn_last_error().decode()


def test_likelihood_of_no_rows():
    lib = _native.load()
    assert lib.bn_states_log_likelihood(0, None, 0, 4, 4, None, None, 8, None, None, None) == 0
    assert _gradient(rows=0, logits=None, s=None, gradient=None) == 0
    assert lib.bn_states_log_likelihood(0, A, 3, 4, 4, None, B, 8, None, None, None) == -1


def _set(tensors):
    """tensors: (dtype, size, address, output address)"""
    lib = _native.load()
    n = len(tensors)
    handle = ctypes.c_void_p()
    rc = lib.bn_gradient_set_create(
        n, _native.i32_array([t[0] for t in tensors]), (ctypes.c_int64 * max(n, 1))(*[t[1] for t in tensors]),
        (ctypes.c_void_p * max(n, 1))(*[t[2] for t in tensors]), (ctypes.c_void_p * max(n, 1))(*[t[3] for t in tensors]),
        ctypes.byref(handle))
    return rc, lib.bn_last_error().decode()


@pytest.mark.parametrize("tensors,message", [
    ([(5, 4, A, B)], "dtype"),
    ([(0, -1, A, B)], "size"),
    ([(0, 4, None, B)], "null"),
    ([(0, 4, A, None)], "null"),
    ([(0, 4, A + 2, B)], "aligned"),
    ([(1, 4, A, B + 4)], "aligned"),
    ([(0, 4, A, A), (0, 4, A, A)], "share memory"),  # one tensor twice, in place
    ([(0, 4, A, B), (0, 4, A + 64, B + 12)], "share memory"),
    ([(0, 4, A, A + 4)], "lies over"),  # shifted over itself
    ([(0, 4, A, A + 64), (0, 4, A + 64, B)], "lies over"),  # over another gradient
    ([(0, 64, A, B), (0, 4, A + 16, A + 16)], "lies over"),
])
def test_gradient_set_refusals(tensors, message):
    rc, error = _set(tensors)
    assert rc == -1 and message in error


def test_gradient_set_calls_check_their_arguments():
    lib = _native.load()
    assert lib.bn_gradient_set_create(1, None, None, None, None, None) == -1
    assert lib.bn_gradient_set_workspace_bytes(None) == -1
    assert lib.bn_gradient_set_norm(None, B, B, None) == -1
    assert lib.bn_gradient_set_clip(None, 1.0, B, B, None) == -1
    assert lib.bn_gradient_set_destroy(None) == 0


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_loads_stay_inside_their_rows(tmp_path):
    """The arithmetic of draw_states' loads, on the host: a padded row may be the last thing in its buffer."""
    source = os.path.join(os.path.dirname(os.path.abspath(__file__)), "row_loads_check.cpp")
    program = str(tmp_path / "row_loads_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", program, source], check=True)
    subprocess.run([program], check=True)


@pytest.mark.parametrize("change", [
    dict(stride=9, g_stride=9, gradient=A + 3 * 4), dict(stride=9, g_stride=9, gradient=A + 6 * 4),
    dict(stride=9, g_stride=9, gradient=A + (9 + 8) * 4), dict(stride=9, g_stride=9, logits=A + 6 * 4, gradient=A),
    dict(stride=9, g_stride=10, gradient=A + 4 * 4), dict(stride=7, g_stride=7, gradient=A + 4 * 4),
    dict(stride=9, g_stride=9, logits=A + 3 * 4, gradient=A),
])
def test_gradient_columns_that_meet_the_logits(change):
    assert _gradient(**change) == -1
    assert "lies over" in _native.load().bn_last_error().decode()
