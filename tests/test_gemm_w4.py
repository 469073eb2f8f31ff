"""Products with 4-bit weights without a GPU: what the C ABI refuses, and what a call would launch."""

from __future__ import annotations

import ctypes

import pytest

from hc import cuda

A, Q, S, Z, C = (0x100000000 * (i + 1) for i in range(5))  # device addresses: inspected only
OK, INVALID, UNSUPPORTED = 0, 1, 2


def plan(m=4, n=1000, k=512, group=128, dtype=cuda.BF16, **change):
    groups = -(-k // group) if group > 0 else 1
    args = cuda._GemmW4Args(m, n, k, dtype, cuda.C_F32, A, max(k, 1), Q, max((k + 1) // 2, 1), S, max(groups, 1), Z,
                            max(groups, 1), group, C, max(n, 1))
    for name, value in change.items():
        setattr(args, name, value)
    info = cuda._OperatorPlanInfo()
    status = cuda.library().hcCudaGemmW4Plan(ctypes.byref(args), 148, ctypes.byref(info))
    return status, info, cuda.library().hcCudaContextLastError(None).decode()


def test_plans() -> None:
    status, info, _ = plan()
    assert (status, info.kernel_launches, info.pieces) == (OK, 1, 1) and info.scratch_bytes > 0
    assert plan(zeros=None)[0] == OK
    assert plan(lda=513)[1].kernel_launches == 2 and plan(a=A + 2)[1].kernel_launches == 2  # one repack of A
    assert plan(k=513)[1].kernel_launches == 2 and plan(m=1, k=513)[1].kernel_launches == 1  # one row has no pitch
    assert plan(m=1, a=A + 2)[1].kernel_launches == 2
    assert plan(q=Q + 1)[1].kernel_launches == 1 and plan(ldq=257)[1].kernel_launches == 1   # q stays where it is
    for group in (32, 64, 128, 256, 384, 4096):
        assert plan(k=4096, group=group)[0] == OK
    for empty in ({"m": 0}, {"n": 0}):
        status, info, _ = plan(a=None, q=None, c=None, scales=None, **empty)
        assert (status, info.kernel_launches) == (OK, 0)
    assert plan(k=0, a=None, q=None, scales=None, zeros=None)[0] == OK
    assert plan(m=64)[0] == OK and plan(c_dtype=cuda.C_BF16)[0] == OK


@pytest.mark.parametrize("change, status, text", [
    ({"m": -1}, INVALID, "m, n, k must be non-negative"),
    ({"m": 65}, UNSUPPORTED, "m <= 64"),
    ({"n": (1 << 30) + 1}, UNSUPPORTED, "at most 2^30"),
    ({"n": 1 << 30, "k": 1 << 30, "lda": 1 << 30, "ldq": 1 << 29, "lds": 1 << 23, "ldz": 1 << 23, "ldc": 1 << 30,
      "a": 1 << 62, "q": 1 << 63, "scales": 1 << 60, "zeros": 1 << 61, "c": 4096}, UNSUPPORTED, "too large"),
    ({"dtype": cuda.F8E4M3}, INVALID, "dtype"),
    ({"c_dtype": cuda.C_F16}, INVALID, "c_dtype"),
    ({"group": 0}, INVALID, "group"),
    ({"group": 16}, INVALID, "group"),
    ({"group": 96}, INVALID, "group"),
    ({"group": 200}, INVALID, "group"),
    ({"group": -128}, INVALID, "group"),
    ({"a": None}, INVALID, "a must not be null"),
    ({"q": None}, INVALID, "q must not be null"),
    ({"scales": None}, INVALID, "scales must not be null"),
    ({"c": None}, INVALID, "c must not be null"),
    ({"a": A + 1}, INVALID, "a must be 2-byte aligned"),
    ({"scales": S + 1}, INVALID, "scales must be 2-byte aligned"),
    ({"c": C + 2}, INVALID, "c must be 4-byte aligned"),
    ({"lda": 511}, INVALID, "pitch of a"),
    ({"ldq": 255}, INVALID, "pitch of q"),
    ({"lds": 3}, INVALID, "pitch of scales"),
    ({"ldz": 3}, INVALID, "pitch of zeros"),
    ({"ldc": 999}, INVALID, "pitch of c"),
    ({"c": A}, INVALID, "c must not overlap a"),
    ({"c": Q + 4}, INVALID, "c must not overlap q"),
    ({"c": S}, INVALID, "c must not overlap scales"),
    ({"c": Z}, INVALID, "c must not overlap zeros"),
])
def test_refusals(change, status, text) -> None:
    got, _, message = plan(**change)
    assert got == status and text in message, message


def test_null_arguments() -> None:
    lib = cuda.library()
    assert lib.hcCudaGemmW4(None, None) == INVALID and lib.hcCudaGemmW4Plan(None, 148, None) == INVALID
    info = cuda._OperatorPlanInfo()
    assert lib.hcCudaGemmW4Plan(None, 148, ctypes.byref(info)) == INVALID
