"""Products with 4-bit weights on a B200 against the definition in 64 bits.

Tolerance. (q - z) a is exact in float32: 5 bits times at most 11. A group's sum passes k / 16 tensor-core
additions, each cutting at most 2^-22 of what it adds; then one product with the scale and one addition per
group, the two halves, and the parts of a split block, 2^-24 each. Together at most (k / 16 + groups + 64)
2^-22 sum |s (q - z) a|, and half a step of C's type for the result.
"""

from __future__ import annotations

import numpy as np
import pytest

from conftest import np_dtype
from hc import cuda
from hc.errors import DeviceError

pytestmark = pytest.mark.gpu

HALF_STEP = {"float32": 2.0**-24, "float16": 2.0**-11, "bfloat16": 2.0**-8}
TINY = {"float32": 2.0**-149, "float16": 2.0**-25, "bfloat16": 2.0**-133}


def empty(ctx, shape, dtype, ld=None) -> cuda.DeviceBuffer:
    buf = cuda.DeviceBuffer(ctx, shape, dtype, ld=ld)
    if buf.nbytes:
        buf.fill_bytes(0xFF)
    return buf


def make(ctx, array, ld=None) -> cuda.DeviceBuffer:
    buf = empty(ctx, array.shape, array.dtype, ld)
    buf.copy_from_host(array)
    return buf


def inputs(m, n, k, group, dtype, zeros=True, seed=1):
    rng = np.random.default_rng([m, n, k, group, seed])
    t = np_dtype(dtype)
    groups = -(-k // group)
    a = rng.standard_normal((m, k)).astype(t)
    q = rng.integers(0, 256, (n, (k + 1) // 2), dtype=np.uint8)
    scales = (0.01 * (0.5 + rng.random((n, groups)))).astype(t)
    z = rng.integers(0, 16, (n, groups), dtype=np.uint8) if zeros else None
    return a, q, scales, z


def weights(q, scales, z, k, group):
    n = q.shape[0]
    digits = np.empty((n, 2 * q.shape[1]))
    digits[:, 0::2], digits[:, 1::2] = q & 15, q >> 4
    at = np.arange(k) // group
    zero = 8.0 if z is None else z.astype(np.float64)[:, at]
    return scales.astype(np.float64)[:, at] * (digits[:, :k] - zero)


def check(got, a, q, scales, z, group) -> None:
    k = a.shape[1]
    w = weights(q, scales, z, k, group)
    a64 = a.astype(np.float64)
    want, size = a64 @ w.T, np.abs(a64) @ np.abs(w).T
    name = got.dtype.name
    bound = HALF_STEP[name] * np.abs(want) + (k / 16 + scales.shape[1] + 64) * 2.0**-22 * size + TINY[name]
    diff = np.abs(got.astype(np.float64) - want)
    assert (diff <= bound).all(), (float((diff / bound).max()), np.argwhere(~(diff <= bound))[:5])


def run(ctx, a, q, scales, z, group, out, pad_a=0, pad_q=0, pad_s=0, pad_c=0):
    m, k = a.shape
    n = q.shape[0]
    ba, bq = make(ctx, a, k + pad_a), make(ctx, q, q.shape[1] + pad_q)
    bs = make(ctx, scales, scales.shape[1] + pad_s)
    bz = None if z is None else make(ctx, z, z.shape[1] + pad_s)
    guard = empty(ctx, (m, n + pad_c), out)
    guard.fill_bytes(0x5A)
    bc = guard.window(0, m, 0, n)
    ctx.gemm_w4(ba, bq, bs, bc, group=group, zeros=bz)
    ctx.synchronize()
    whole = guard.to_numpy()
    assert (np.ascontiguousarray(whole[:, n:]).view(np.uint8) == 0x5A).all()  # nothing beside C is written
    return np.ascontiguousarray(whole[:, :n])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("m, n, k, group", [
    (1, 1, 1, 32), (1, 1, 2, 128), (3, 5, 31, 32), (1, 127, 33, 32), (8, 128, 255, 64), (2, 129, 256, 128),
    (5, 300, 257, 32), (7, 1031, 1000, 64), (9, 257, 700, 128), (16, 500, 2048, 32), (17, 130, 1030, 64),
    (33, 200, 513, 128), (64, 640, 1536, 128), (64, 77, 91, 32), (1, 4096, 4096, 128), (4, 16, 16384, 64)])
def test_products(m, n, k, group, dtype, gpu_ctx) -> None:
    for zeros in (True, False):
        a, q, scales, z = inputs(m, n, k, group, dtype, zeros)
        check(run(gpu_ctx, a, q, scales, z, group, np_dtype(dtype)), a, q, scales, z, group)
    check(run(gpu_ctx, a, q, scales, z, group, np.float32), a, q, scales, z, group)


@pytest.mark.parametrize("group", [256, 384, 1024, 4096])
def test_long_groups(group, gpu_ctx) -> None:
    a, q, scales, z = inputs(3, 200, 2100, group, "float16")
    check(run(gpu_ctx, a, q, scales, z, group, np.float32), a, q, scales, z, group)


@pytest.mark.parametrize("pad_a, pad_q, pad_s, pad_c", [(8, 16, 0, 0), (1, 0, 3, 5), (0, 1, 1, 1), (3, 4, 0, 2), (0, 15, 2, 0)])
@pytest.mark.parametrize("m", [2, 12, 40])
def test_pitches(m, pad_a, pad_q, pad_s, pad_c, gpu_ctx) -> None:
    a, q, scales, z = inputs(m, 301, 992, 64, "bfloat16", seed=2)
    got = run(gpu_ctx, a, q, scales, z, 64, np.float32, pad_a, pad_q, pad_s, pad_c)
    check(got, a, q, scales, z, 64)
    # Where things lie does not change a bit.
    assert np.array_equal(got, run(gpu_ctx, a, q, scales, z, 64, np.float32))


@pytest.mark.parametrize("offset", [1, 2, 4, 8, 15])
def test_weights_that_start_anywhere(offset, gpu_ctx) -> None:
    """q as a window of a larger buffer, at every kind of byte offset."""
    a, q, scales, z = inputs(2, 140, 640, 128, "float16", seed=3)
    big = empty(gpu_ctx, (140, 512), np.uint8)
    host = np.random.default_rng(4).integers(0, 256, (140, 512), dtype=np.uint8)
    host[:, offset:offset + q.shape[1]] = q
    big.copy_from_host(host)
    bc = empty(gpu_ctx, (2, 140), np.float32)
    gpu_ctx.gemm_w4(make(gpu_ctx, a), big.window(0, 140, offset, offset + q.shape[1]), make(gpu_ctx, scales), bc, group=128,
                    zeros=make(gpu_ctx, z))
    gpu_ctx.synchronize()
    check(bc.to_numpy(), a, q, scales, z, 128)


def test_repeats_bit_for_bit_and_rows_are_independent(gpu_ctx) -> None:
    a, q, scales, z = inputs(8, 1500, 3000, 64, "bfloat16", seed=5)
    first = run(gpu_ctx, a, q, scales, z, 64, np.float32)
    for _ in range(3):
        assert np.array_equal(first, run(gpu_ctx, a, q, scales, z, 64, np.float32))
    for m in (1, 5):
        assert np.array_equal(first[:m], run(gpu_ctx, a[:m], q, scales, z, 64, np.float32))


def test_non_finite_activations_stay_in_their_row(gpu_ctx) -> None:
    a, q, scales, z = inputs(4, 150, 300, 32, "float16", seed=6)
    a[1, 7], a[2, 299] = np.nan, np.inf
    got = run(gpu_ctx, a, q, scales, z, 32, np.float32)
    good = [0, 3]
    check(got[good], a[good], q, scales, z, 32)
    assert np.isnan(got[1]).all() and not np.isfinite(got[2]).any()


def test_extreme_scales(gpu_ctx) -> None:
    """Scales at both ends of bfloat16's range: they meet float32 sums, not 16-bit weights."""
    a, q, scales, z = inputs(2, 64, 256, 128, "bfloat16", seed=7)
    scales = (scales.astype(np.float64) * np.where(np.arange(64) % 2, 1e30, 1e-30)[:, None]).astype(scales.dtype)
    check(run(gpu_ctx, a, q, scales, z, 128, np.float32), a, q, scales, z, 128)


def test_more_units_than_ctas_and_fewer(gpu_ctx) -> None:
    for m, n, k in ((1, 40000, 512), (1, 64, 512), (10, 20000, 1024), (1, 128, 65536), (40, 20000, 700)):
        a, q, scales, z = inputs(m, n, k, 128, "float16", seed=8)
        check(run(gpu_ctx, a, q, scales, z, 128, np.float32), a, q, scales, z, 128)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m, n, k", [(17, 20000, 1024), (64, 20001, 1024), (64, 20000, 999), (30, 9, 8000), (64, 1500, 5000)])
def test_blocks_whole_and_shared(m, n, k, group, gpu_ctx) -> None:
    """CTAs that begin and end inside row blocks with whole ones between, and blocks shared by many."""
    a, q, scales, z = inputs(m, n, k, group, "bfloat16", seed=9)
    got = run(gpu_ctx, a, q, scales, z, group, np_dtype("bfloat16"))
    check(got, a, q, scales, z, group)
    assert np.array_equal(got, run(gpu_ctx, a, q, scales, z, group, np_dtype("bfloat16")))


def test_empty_products(gpu_ctx) -> None:
    c = empty(gpu_ctx, (3, 5), np.float32)
    gpu_ctx.gemm_w4(cuda.DeviceBuffer(gpu_ctx, (3, 0), np.float16), cuda.DeviceBuffer(gpu_ctx, (5, 0), np.uint8),
                    cuda.DeviceBuffer(gpu_ctx, (5, 0), np.float16), c, group=32)
    gpu_ctx.synchronize()
    assert (c.to_numpy() == 0).all()
    none = cuda.DeviceBuffer(gpu_ctx, (0, 64), np.float16)
    q, s = empty(gpu_ctx, (5, 32), np.uint8), empty(gpu_ctx, (5, 2), np.float16)
    gpu_ctx.gemm_w4(none, q, s, cuda.DeviceBuffer(gpu_ctx, (0, 5), np.float16), group=32)
    gpu_ctx.synchronize()


def test_refusals_reach_python(gpu_ctx) -> None:
    a, q = empty(gpu_ctx, (4, 64), np.float16), empty(gpu_ctx, (9, 32), np.uint8)
    s, c = empty(gpu_ctx, (9, 2), np.float16), empty(gpu_ctx, (4, 9), np.float32)
    with pytest.raises(ValueError, match="q as uint8"):
        gpu_ctx.gemm_w4(a, empty(gpu_ctx, (9, 31), np.uint8), s, c, group=32)
    with pytest.raises(ValueError, match="scales must be float16"):
        gpu_ctx.gemm_w4(a, q, s, c, group=64)
    with pytest.raises(ValueError, match="zeros must be uint8"):
        gpu_ctx.gemm_w4(a, q, s, c, group=32, zeros=s)
    with pytest.raises(DeviceError, match="group must be"):
        gpu_ctx.gemm_w4(a, q, empty(gpu_ctx, (9, 4), np.float16), c, group=16)
    with pytest.raises(DeviceError, match="m <= 64"):
        gpu_ctx.gemm_w4(empty(gpu_ctx, (65, 64), np.float16), q, s, empty(gpu_ctx, (65, 9), np.float32), group=32)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("pad_q", [0, 1])
def test_zero_points_beyond_fifteen(pad_q, group, dtype, gpu_ctx) -> None:
    """0..63 are zero points, of a larger byte the low six bits, whatever the number of rows of A."""
    for m in (1, 9, 16, 17, 40):
        a, q, scales, _ = inputs(m, 150, 640, group, dtype, seed=10)
        z = np.random.default_rng(group).integers(0, 64, (150, 640 // group), dtype=np.uint8)
        z[:, 0] = np.arange(150) % 64
        got = run(gpu_ctx, a, q, scales, z, group, np.float32, pad_q=pad_q)
        check(got, a, q, scales, z, group)
        assert np.array_equal(got, run(gpu_ctx, a, q, scales, z + np.uint8(64 * (m % 4)), group, np.float32, pad_q=pad_q))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("m, group, k", [(1, 128, 8192), (3, 64, 8192), (8, 64, 8192), (16, 32, 8192), (8, 128, 8191), (32, 64, 8192),
                                         (64, 128, 8192)])
def test_long_products_stay_right_in_every_column(m, group, k, dtype, gpu_ctx) -> None:
    """Rings that are refilled some hundred times by every CTA: no stage is overwritten while its last words are being
    read. The weights are one block of rows a hundred times over, so that the definition is computed once."""
    block, copies = 1000, 100
    a, q, scales, z = inputs(m, block, k, group, dtype, seed=11)
    many = [empty(gpu_ctx, (block * copies, v.shape[1]), v.dtype) for v in (q, scales, z)]
    for buf, v in zip(many, (q, scales, z)):
        for i in range(copies):
            buf.window(i * block, (i + 1) * block, 0, v.shape[1]).copy_from_host(v)
    ba, c = make(gpu_ctx, a), empty(gpu_ctx, (m, block * copies), np.float32)
    first = None
    for _ in range(3):
        c.fill_bytes(0xFF)
        gpu_ctx.gemm_w4(ba, many[0], many[1], c, group=group, zeros=many[2])
        gpu_ctx.synchronize()
        got = c.to_numpy()
        assert first is None or np.array_equal(got, first)
        first = got
    w = weights(q, scales, z, k, group)
    a64 = a.astype(np.float64)
    want, size = a64 @ w.T, np.abs(a64) @ np.abs(w).T
    bound = HALF_STEP["float32"] * np.abs(want) + (k / 16 + scales.shape[1] + 64) * 2.0**-22 * size
    # (A stage's last words taken from the next stage are off by 1e-4 to 1e-3 of the sum of sizes; the bound is 2e-4.)
    assert (np.abs(got.reshape(m, copies, block) - want[:, None]) <= bound[:, None]).all()


@pytest.mark.parametrize("dtype, out", [("float16", "float16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("m", [1, 7, 16, 40])
def test_everything_at_odd_places(m, dtype, out, gpu_ctx) -> None:
    """All matrices as windows that begin inside a row of a larger buffer, whose other columns stay as they are."""
    n, k, group = 261, 1100, 64
    a, q, scales, z = inputs(m, n, k, group, dtype, seed=12)
    whole_buffers = []  # (a window does not keep the buffer it lies in)

    def window(values, left, pad):
        host = np.zeros((values.shape[0], left + values.shape[1] + pad), values.dtype)
        host.view(np.uint8)[:] = 0x5A
        host[:, left:left + values.shape[1]] = values
        whole_buffers.append(make(gpu_ctx, host))
        return whole_buffers[-1].window(0, values.shape[0], left, left + values.shape[1])

    guard = empty(gpu_ctx, (m, n + 5), np_dtype(out))
    guard.fill_bytes(0x5A)
    parts = [window(v, left, pad) for v, left, pad in ((a, 3, 2), (q, 5, 1), (scales, 1, 1), (z, 3, 4))]
    gpu_ctx.gemm_w4(parts[0], parts[1], parts[2], guard.window(0, m, 3, n + 3), group=group, zeros=parts[3])
    gpu_ctx.synchronize()
    whole = guard.to_numpy()
    check(np.ascontiguousarray(whole[:, 3:n + 3]), a, q, scales, z, group)
    for beside in (whole[:, :3], whole[:, n + 3:]):
        assert (np.ascontiguousarray(beside).view(np.uint8) == 0x5A).all()
