"""A 16-bit C whose rows end inside a 32-bit word, with pitches that TMA can address: what lies beside C stays."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import np_dtype
from hc import cuda

pytestmark = pytest.mark.gpu

HALF_STEP = {"float16": 2.0**-11, "bfloat16": 2.0**-8}


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("epilogue", [(), (("scale", 0.5), ("max", 0.0))])
@pytest.mark.parametrize("m, n, k", [(8, 1031, 512), (40, 77, 300), (100, 301, 128), (128, 259, 700), (300, 1001, 96), (256, 257, 8192),
                                     (1024, 1029, 512), (2048, 1537, 4096), (6000, 4093, 4100)])
def test_nothing_beside_an_odd_row_is_written(m, n, k, epilogue, dtype, gpu_ctx) -> None:
    rng = np.random.default_rng([m, n, k])
    t = np_dtype(dtype)
    a = (rng.standard_normal((m, k), dtype=np.float32) / np.sqrt(k)).astype(t)
    b = rng.standard_normal((k, n), dtype=np.float32).astype(t)
    ba, bb = gpu_ctx.to_device(a), gpu_ctx.to_device(b)
    ld = (n + 7) // 8 * 8
    for left in (0, 8):
        whole = cuda.DeviceBuffer(gpu_ctx, (m, left + ld + 8), t)
        whole.fill_bytes(0x5A)
        gpu_ctx.gemm(ba, bb, whole.window(0, m, left, left + n), epilogue=epilogue)
        gpu_ctx.synchronize()
        out = whole.to_numpy()
        for beside in (out[:, :left], out[:, left + n:]):
            assert (np.ascontiguousarray(beside).view(np.uint8) == 0x5A).all()
        rows = np.unique(np.linspace(0, m - 1, 60).astype(int))
        want = a[rows].astype(np.float64) @ b.astype(np.float64)
        size = np.abs(a[rows].astype(np.float64)) @ np.abs(b.astype(np.float64))
        if epilogue:
            want, size = np.maximum(0.5 * want, 0.0), 0.5 * size
        # The tensor cores cut at most 2^-22 of what they add, 16 of k at a time; one rounding of the result.
        bound = HALF_STEP[dtype] * np.abs(want) + (k / 16 + 16) * 2.0**-22 * size + 2.0**-25
        assert (np.abs(out[rows, left:left + n].astype(np.float64) - want) <= bound).all()
