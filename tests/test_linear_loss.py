"""The linear cross entropy without a GPU: what the C ABI refuses, and what a call would launch."""

from __future__ import annotations

import ctypes

import pytest

from hc import cuda

# Integers standing for device addresses, far enough apart for every size below.
H, W, T, LOSS, LSE, DLOSS, DH, DW = (0x100000000 * (i + 1) for i in range(8))
OK, INVALID, UNSUPPORTED = 0, 1, 2


def _call(struct, entry, values, change):
    args = struct(*values)
    for name, value in change.items():
        setattr(args, name, value)
    info = cuda._OperatorPlanInfo()
    status = getattr(cuda.library(), entry)(ctypes.byref(args), 148, ctypes.byref(info))
    return status, info, cuda.library().hcCudaContextLastError(None).decode()


def forward(rows=100, vocab=1000, width=64, dtype=cuda.BF16, **change):
    return _call(cuda._LinearLossArgs, "hcCudaLinearLossPlan",
                 (rows, vocab, width, dtype, 1, H, width, W, width, T, -100, LOSS, LSE), change)


def backward(rows=100, vocab=1000, width=64, dtype=cuda.BF16, **change):
    return _call(cuda._LinearLossBackwardArgs, "hcCudaLinearLossBackwardPlan",
                 (rows, vocab, width, dtype, 1, H, width, W, width, T, -100, LSE, DLOSS, DH, width, DW, width), change)


def test_forward_plans() -> None:
    status, info, _ = forward()
    assert (status, info.kernel_launches, info.pieces) == (OK, 2, 1)
    assert info.scratch_bytes >= 100 * 8 * 8  # eight half tiles of two floats per row
    assert forward(width=65)[1].kernel_launches == 3          # odd pitches: one repack
    assert forward(ldh=72, ldw=72)[1].kernel_launches == 2
    assert forward(h=H + 2)[1].kernel_launches == 3
    status, info, _ = forward(rows=0, h=None, targets=None, loss=None, lse=None)
    assert (status, info.kernel_launches) == (OK, 0)


def test_the_logits_are_never_held(monkeypatch) -> None:
    """The scratch of both passes stays far below the logits' bytes, and g's piece within its bound."""
    rows, vocab, width = 65536, 131072, 4096
    status, info, _ = forward(rows, vocab, width)
    assert status == OK and info.scratch_bytes < rows * vocab * 4 // 60
    status, info, _ = backward(rows, vocab, width)
    assert status == OK and info.pieces == 64
    assert info.scratch_bytes <= (1 << 29) + rows * width * (4 + 2) + (64 << 20)
    monkeypatch.setenv("HC_CUDA_LOSS_PIECE", "512")
    assert backward()[1].pieces == 2 and backward(vocab=1025)[1].pieces == 3


def test_backward_plans() -> None:
    status, info, _ = backward()
    # The scales with h's rows, the logits, two products, and dh rounded from the float32 of its clusters.
    assert (status, info.pieces, info.kernel_launches) == (OK, 1, 5)
    assert backward(dw=None)[1].kernel_launches == 4 and backward(dh=None)[1].kernel_launches == 3
    assert backward(dh=None, dw=None)[1].kernel_launches == 0
    assert backward(dtype=cuda.F16)[1].kernel_launches == 5
    assert backward(8192, 2048, 2048)[1].kernel_launches == 4  # a product of many tiles writes dh at once
    status, info, _ = backward(rows=0, h=None, targets=None, lse=None, dloss=None)
    assert (status, info.kernel_launches) == (OK, 0)


COMMON = [
    ({"rows": -1}, INVALID, "rows must be non-negative"),
    ({"vocab": 0}, INVALID, "vocab and width at least 1"),
    ({"width": 0}, INVALID, "vocab and width at least 1"),
    ({"rows": (1 << 30) + 1}, UNSUPPORTED, "at most 2^30"),
    ({"rows": 1 << 30, "vocab": 1 << 30}, UNSUPPORTED, "too many tiles"),
    ({"dtype": cuda.F8E4M3}, INVALID, "dtype must be HC_CUDA_F16 or HC_CUDA_BF16"),
    ({"targets_64": 2}, INVALID, "targets_64"),
    ({"h": None}, INVALID, "h must not be null"),
    ({"w": W + 1}, INVALID, "w must be 2-byte aligned"),
    ({"targets": T + 4}, INVALID, "targets must be 8-byte aligned"),
    ({"targets": None}, INVALID, "targets must not be null"),
    ({"ldh": 63}, INVALID, "pitch of h"),
    ({"ldw": 63}, INVALID, "pitch of w"),
    ({"lse": None}, INVALID, "lse must not be null"),
]


@pytest.mark.parametrize("change, status, text", COMMON + [
    ({"loss": None}, INVALID, "loss must not be null"),
    ({"loss": LSE}, INVALID, "loss must not overlap lse"),
    ({"loss": H}, INVALID, "loss must not overlap h"),
    ({"lse": W + 4}, INVALID, "lse must not overlap w"),
    ({"lse": T}, INVALID, "lse must not overlap targets"),
])
def test_forward_refusals(change, status, text) -> None:
    got, _, message = forward(**change)
    assert got == status and text in message, message


@pytest.mark.parametrize("change, status, text", COMMON + [
    ({"dloss": None}, INVALID, "dloss must not be null"),
    ({"lddh": 63}, INVALID, "pitch of dh"),
    ({"lddw": 63}, INVALID, "pitch of dw"),
    ({"dh": DH + 1}, INVALID, "dh must be 2-byte aligned"),
    ({"dh": H}, INVALID, "dh must not overlap h"),
    ({"dw": W}, INVALID, "dw must not overlap w"),
    ({"dw": DH}, INVALID, "dh must not overlap dw"),
    ({"dh": LSE}, INVALID, "dh must not overlap lse"),
])
def test_backward_refusals(change, status, text) -> None:
    got, _, message = backward(**change)
    assert got == status and text in message, message


def test_null_arguments() -> None:
    lib = cuda.library()
    info = cuda._OperatorPlanInfo()
    for name in ("hcCudaLinearLoss", "hcCudaLinearLossBackward"):
        assert getattr(lib, name)(None, None) == INVALID
        assert getattr(lib, name + "Plan")(None, 148, ctypes.byref(info)) == INVALID
        assert getattr(lib, name + "Plan")(None, 148, None) == INVALID


@pytest.mark.parametrize("address", [1 << 40, (1 << 40) + 0x20000, (1 << 40) + 2, (1 << 40) - 0x1000])
def test_gradients_may_lie_at_any_address(address) -> None:
    """The plan is made before the scratch exists: no address of the caller's is mistaken for it."""
    for change in ({"dw": address}, {"dh": address}, {"w": address}, {"h": address}):
        status, info, message = backward(**change)
        assert status == OK and info.kernel_launches > 0, message
    assert backward(dw=address, dh=address)[0] == INVALID  # overlaps among the caller's own are still found


def test_an_ignore_index_is_passed_on_as_it_is_or_refused() -> None:
    """The C ABI takes 64 bits; a larger number would arrive as another, possibly a token's."""
    h, w = cuda.DeviceBuffer.wrap(None, H, (4, 8), "bfloat16"), cuda.DeviceBuffer.wrap(None, W, (9, 8), "bfloat16")
    targets = cuda.DeviceBuffer.wrap(None, T, (4,), "int64")
    for index in (-100, 0, 8, -(1 << 63), (1 << 63) - 1):
        args = cuda._LinearLossArgs(*cuda.Context._loss_call("linear_cross_entropy", h, w, targets, index), LOSS, LSE)
        assert args.ignore_index == index
    for index in ((1 << 64) + 5, 1 << 63, -(1 << 63) - 1):
        with pytest.raises(ValueError, match="64-bit"):
            cuda.Context._loss_call("linear_cross_entropy", h, w, targets, index)
