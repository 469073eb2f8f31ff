"""Layer norm without a GPU: what the C ABI refuses, and what a call would launch. The checks are those
of the computing entry points; the plan calls run them without a device."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from hc import cuda

# Integers standing for device addresses: inspected, never dereferenced.
X, Y, W, B, MEAN, RSTD, DY, DX, DW, DB = (0x10000000 * (i + 1) for i in range(10))
OK, INVALID, UNSUPPORTED = 0, 1, 2


def forward(rows=10, cols=64, dtype=cuda.C_BF16, param=cuda.C_BF16, **change):
    args = cuda._LayerNormArgs(rows, cols, dtype, param, X, cols, W, B, Y, cols, MEAN, RSTD, 1e-5)
    for name, value in change.items():
        setattr(args, name, value)
    info = cuda._OperatorPlanInfo()
    status = cuda.library().hcCudaLayerNormPlan(ctypes.byref(args), 148, ctypes.byref(info))
    return status, info, cuda.library().hcCudaContextLastError(None).decode()


def backward(rows=10, cols=64, dtype=cuda.C_BF16, param=cuda.C_BF16, **change):
    args = cuda._LayerNormBackwardArgs(rows, cols, dtype, param, DY, cols, X, cols, W, MEAN, RSTD, DX, cols, DW, DB)
    for name, value in change.items():
        setattr(args, name, value)
    info = cuda._OperatorPlanInfo()
    status = cuda.library().hcCudaLayerNormBackwardPlan(ctypes.byref(args), 148, ctypes.byref(info))
    return status, info, cuda.library().hcCudaContextLastError(None).decode()


def test_plans() -> None:
    status, info, _ = forward()
    assert (status, info.kernel_launches, info.scratch_bytes) == (OK, 1, 0)
    for empty in ({"rows": 0}, {"cols": 0}):
        status, info, _ = forward(x=None, y=None, **empty)
        assert (status, info.kernel_launches) == (OK, 0)
    status, info, _ = backward(rows=16384, cols=4096)
    assert status == OK and info.kernel_launches == 2 and info.scratch_bytes > 0
    status, info, _ = backward(rows=16384, cols=4096, dweight=None, dbias=None)
    assert status == OK and info.kernel_launches == 1 and info.scratch_bytes == 0
    status, info, _ = backward(rows=7, cols=1 << 20)
    assert status == OK and info.kernel_launches == 3
    status, info, _ = backward(rows=0, x=None, dy=None, dx=None, mean=None, rstd=None)
    assert (status, info.kernel_launches) == (OK, 0)


@pytest.mark.parametrize("change, status, text", [
    ({"rows": -1}, INVALID, "rows and cols"),
    ({"rows": 1 << 31}, UNSUPPORTED, "rows"),
    ({"dtype": 7}, INVALID, "dtype"),
    ({"param_dtype": cuda.C_F16}, INVALID, "param_dtype"),
    ({"eps": -1.0}, INVALID, "eps"),
    ({"eps": float("nan")}, INVALID, "eps"),
    ({"eps": float("inf")}, INVALID, "eps"),
    ({"x": None}, INVALID, "x must not be null"),
    ({"y": None}, INVALID, "y must not be null"),
    ({"x": X + 1}, INVALID, "x must be 2-byte aligned"),
    ({"mean": MEAN + 2}, INVALID, "mean must be 4-byte aligned"),
    ({"ldx": 63}, INVALID, "pitch of x"),
    ({"ldy": 63}, INVALID, "pitch of y"),
    ({"y": X + 2}, INVALID, "y must not partially overlap x"),
    ({"y": X, "ldy": 65}, INVALID, "y must not partially overlap x"),
    ({"y": W}, INVALID, "y must not overlap weight"),
    ({"mean": X}, INVALID, "mean must not overlap x"),
    ({"rstd": MEAN}, INVALID, "mean must not overlap rstd"),
])
def test_forward_refusals(change, status, text) -> None:
    got, _, message = forward(**change)
    assert got == status and text in message, message


@pytest.mark.parametrize("change, status, text", [
    ({"cols": -3}, INVALID, "rows and cols"),
    ({"dtype": -1}, INVALID, "dtype"),
    ({"param_dtype": cuda.C_F16}, INVALID, "param_dtype"),
    ({"mean": None}, INVALID, "mean must not be null"),
    ({"rstd": None}, INVALID, "rstd must not be null"),
    ({"dx": None}, INVALID, "dx must not be null"),
    ({"lddy": 10}, INVALID, "pitch of dy"),
    ({"lddx": 10}, INVALID, "pitch of dx"),
    ({"dx": DY + 4}, INVALID, "dx must not partially overlap dy"),
    ({"dx": W}, INVALID, "dx must not overlap weight"),
    ({"dweight": DB}, INVALID, "dweight must not overlap dbias"),
    ({"dbias": X}, INVALID, "dbias must not overlap x"),
    ({"dweight": W + 2}, INVALID, "dweight must not overlap weight"),
])
def test_backward_refusals(change, status, text) -> None:
    got, _, message = backward(**change)
    assert got == status and text in message, message


def test_in_place_is_allowed() -> None:
    assert forward(y=X)[0] == OK
    assert backward(dx=DY)[0] == OK and backward(dx=X)[0] == OK


def test_null_arguments() -> None:
    lib = cuda.library()
    assert lib.hcCudaLayerNorm(None, None) == INVALID and lib.hcCudaLayerNormBackward(None, None) == INVALID
    assert lib.hcCudaLayerNormPlan(None, 148, None) == INVALID
    info = cuda._OperatorPlanInfo()
    assert lib.hcCudaLayerNormPlan(None, 148, ctypes.byref(info)) == INVALID
    assert lib.hcCudaLayerNormBackwardPlan(None, 148, ctypes.byref(info)) == INVALID


def test_device_buffers_take_type_names() -> None:
    assert cuda.DeviceBuffer.wrap(None, 0, (3, 4), "bfloat16").dtype.name == "bfloat16"
    assert cuda.DeviceBuffer.wrap(None, 0, (3, 4), "float32").dtype == np.float32


@pytest.mark.parametrize("sm_count", [132, 140, 148, 160])
def test_a_plan_is_that_of_the_device_it_is_asked_for(sm_count) -> None:
    """At odd places few rows (of 4 MiB and more) are walked three times and many go through the ring, with launches
    and scratch of their own; where that changes depends on the device, and both change together."""
    def plan(rows):
        args = cuda._LayerNormBackwardArgs(rows, 8191, cuda.C_BF16, cuda.C_BF16, DY, 8191, X, 8191, W, MEAN, RSTD, DX, 8191,
                                           DW, DB)
        info = cuda._OperatorPlanInfo()
        assert cuda.library().hcCudaLayerNormBackwardPlan(ctypes.byref(args), sm_count, ctypes.byref(info)) == OK
        return info.kernel_launches, info.scratch_bytes

    row = 2 * 4 * 8191  # of the partial sums of dweight and dbias
    few, many = plan(2 * sm_count - 1), plan(2 * sm_count)
    column_blocks = -(-8191 // 256)
    assert few == (3, row * -(-8 * sm_count // column_blocks))  # chunks of rows: eight CTAs a multiprocessor
    assert many == (2, row * (sm_count // 8 * 8))               # one CTA a multiprocessor, as many of each of eight places
