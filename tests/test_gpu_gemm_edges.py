"""A C whose rows start on 16-byte boundaries and end inside a 16-byte piece: what lies beside C stays as it was."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import np_dtype
from hc import cuda

pytestmark = pytest.mark.gpu

HALF_STEP = {"float16": 2.0**-11, "bfloat16": 2.0**-8, "float32": 2.0**-24}
# Every form of the product: few rows, narrow and wide tiles, pairs, split and clustered k, 512-row tiles.
SHAPES = [(8, 1024, 512), (40, 72, 300), (100, 304, 128), (128, 256, 700), (300, 1000, 96), (256, 256, 8192), (1024, 1024, 512),
          (2048, 1536, 4096), (6000, 4096, 4100)]


def product(ctx, m, n, k, out, lefts, epilogue=(), accumulate=False):
    rng = np.random.default_rng([m, n, k])
    kind = "bfloat16" if out == "bfloat16" else "float16"
    a = (rng.standard_normal((m, k), dtype=np.float32) / np.sqrt(k)).astype(np_dtype(kind))
    b = rng.standard_normal((k, n), dtype=np.float32).astype(np_dtype(kind))
    ba, bb = ctx.to_device(a), ctx.to_device(b)
    t = np.dtype(np_dtype(out))
    piece = 16 // t.itemsize
    ld = (n + piece - 1) // piece * piece
    for left in lefts:
        host = np.zeros((m, left + ld + 8), t)
        host.view(np.uint8)[:] = 0x5A
        c0 = rng.standard_normal((m, n), dtype=np.float32) if accumulate else None
        if accumulate:
            host[:, left:left + n] = c0
        whole = ctx.to_device(host)
        ctx.gemm(ba, bb, whole.window(0, m, left, left + n), epilogue=epilogue, accumulate=accumulate)
        ctx.synchronize()
        got = whole.to_numpy()
        for beside in (got[:, :left], got[:, left + n:]):
            assert (np.ascontiguousarray(beside).view(np.uint8) == 0x5A).all()
        rows = np.unique(np.linspace(0, m - 1, 60).astype(int))
        want = a[rows].astype(np.float64) @ b.astype(np.float64)
        size = np.abs(a[rows].astype(np.float64)) @ np.abs(b.astype(np.float64))
        if accumulate:
            want, size = want + c0[rows], size + np.abs(c0[rows])
        if epilogue:
            want, size = np.maximum(0.5 * want, 0.0), 0.5 * size
        # The tensor cores cut at most 2^-22 of what they add, 16 of k at a time; one rounding of the result.
        bound = HALF_STEP[out] * np.abs(want) + (k / 16 + 16) * 2.0**-22 * size + 2.0**-25
        assert (np.abs(got[rows, left:left + n].astype(np.float64) - want) <= bound).all()


@pytest.mark.parametrize("out", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("more", [1, 2, 3, 4, 6])
@pytest.mark.parametrize("m, n, k", SHAPES)
def test_nothing_beside_c_is_written(m, n, k, more, out, gpu_ctx) -> None:
    if m * n > 1 << 21 and more not in (1, 4):
        more = 2
    product(gpu_ctx, m, n + more, k, out, (0, 8))


@pytest.mark.parametrize("more", [1, 2, 3])
@pytest.mark.parametrize("m, n, k", SHAPES[:8])
def test_nothing_beside_c_is_written_by_fused_work(m, n, k, more, gpu_ctx) -> None:
    product(gpu_ctx, m, n + more, k, "float32", (0,), (("scale", 0.5), ("max", 0.0)))
    product(gpu_ctx, m, n + more, k, "float32", (4,), (), accumulate=True)
    product(gpu_ctx, m, n + more, k, "float32", (0,), (("scale", 0.5), ("max", 0.0)), accumulate=True)
    product(gpu_ctx, m, n + more, k, "float16", (8,), (("scale", 0.5), ("max", 0.0)))


@pytest.mark.parametrize("m, n, k", [(100, 301, 128), (256, 258, 8192), (1030, 2051, 600), (2500, 2503, 2000)])
def test_host_arrays_keep_what_lies_beside_c(m, n, k, gpu_ctx) -> None:
    """The host-buffer call stages C with rows of its own, which TMA may fill up."""
    rng = np.random.default_rng([m, n, k])
    a = (rng.standard_normal((m, k), dtype=np.float32) / np.sqrt(k)).astype(np.float16)
    b = rng.standard_normal((k, n), dtype=np.float32).astype(np.float16)
    host = np.full((m, n + 5), 7.0, np.float32)
    gpu_ctx.gemm_host(a, b, host[:, :n])
    assert (host[:, n:] == 7.0).all()
    want = a.astype(np.float64) @ b.astype(np.float64)
    size = np.abs(a.astype(np.float64)) @ np.abs(b.astype(np.float64))
    assert (np.abs(host[:, :n] - want) <= 2.0**-24 * np.abs(want) + (k / 16 + 16) * 2.0**-22 * size).all()
