"""Layer norm and its gradients on a B200 against the formula in 64 bits.

Tolerances. u = 2^-24 is half a float32 step, h half a step of the stored type. A float32 sum of the kernel
is a tree whose depth is at most 65 values per thread, 5 shuffles and 8 more for the warps, and longer only
for rows of more than 32768 values (cols / 1024): DEPTH below bounds it, so a sum of s_i is off by at
most DEPTH u sum|s_i|. Every product, difference and quotient adds u relative. What follows from that is
written at each check; the factor 2 stands for the terms of second order.
"""

from __future__ import annotations

import ctypes
import threading

import numpy as np
import pytest

from conftest import np_dtype
from hc import cuda
from hc.errors import DeviceError

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF_STEP = {"float32": 2.0**-24, "float16": 2.0**-11, "bfloat16": 2.0**-8}
TINY = {"float32": 2.0**-149, "float16": 2.0**-25, "bfloat16": 2.0**-133}  # half the smallest subnormal, or more
EPS = 1e-5


def depth(cols: int) -> float:
    return 2.0 * (64 + cols / 512)


def make(ctx, array: np.ndarray, ld: int | None = None) -> cuda.DeviceBuffer:
    buf = cuda.DeviceBuffer(ctx, array.shape, array.dtype, ld=ld)
    if buf.nbytes:
        buf.fill_bytes(0xFF)  # NaN in the padding: nothing there may count
    buf.copy_from_host(array)
    return buf


def empty(ctx, shape, dtype, ld: int | None = None) -> cuda.DeviceBuffer:
    buf = cuda.DeviceBuffer(ctx, shape, dtype, ld=ld)
    if buf.nbytes:
        buf.fill_bytes(0xFF)
    return buf


def inputs(rows: int, cols: int, dtype: str, param: str, seed: int, offset: float = 0.5):
    rng = np.random.default_rng([rows, cols, seed])
    t, p = np_dtype(dtype), np_dtype(param)
    x = (rng.standard_normal((rows, cols)) * np.exp(0.5 * rng.standard_normal(cols)) + offset).astype(t)
    dy = (0.1 * rng.standard_normal((rows, cols))).astype(t)
    w = (1.0 + 0.1 * rng.standard_normal(cols)).astype(p)
    b = (0.1 * rng.standard_normal(cols)).astype(p)
    return x, dy, w, b


def reference(x, w, b):
    x, w, b = (v.astype(np.float64) for v in (x, w, b))
    mean = x.mean(axis=1)
    rstd = 1.0 / np.sqrt(((x - mean[:, None]) ** 2).mean(axis=1) + EPS)
    n = (x - mean[:, None]) * rstd[:, None]
    return n * w + b, mean, rstd, n


def reference_backward(dy, x, w, mean, rstd):
    dy, x, w, mean, rstd = (v.astype(np.float64) for v in (dy, x, w, mean, rstd))
    n = (x - mean[:, None]) * rstd[:, None]
    a = dy * w
    dx = rstd[:, None] * (a - a.mean(axis=1, keepdims=True) - n * (a * n).mean(axis=1, keepdims=True))
    return dx, (dy * n).sum(axis=0), dy.sum(axis=0), n, a


def check_forward(dtype, x, w, b, y, mean, rstd) -> None:
    cols = x.shape[1]
    d = depth(cols)
    want_y, want_mean, want_rstd, n = reference(x, w, b)
    size = np.abs(x.astype(np.float64)).mean(axis=1)
    mean_err = d * U * size
    assert (np.abs(mean - want_mean) <= mean_err + 1e-45).all()
    # variance: d u relative for its sum, and the square of the mean's error
    var = 1.0 / want_rstd**2 - EPS
    rstd_rel = 0.5 * (d * U * var + mean_err**2) * want_rstd**2 + 8 * U
    assert (np.abs(rstd - want_rstd) <= 2 * rstd_rel * want_rstd).all()
    w64, b64 = np.abs(w.astype(np.float64)), np.abs(b.astype(np.float64))
    err = (w64 * want_rstd[:, None] * mean_err[:, None] + np.abs(n) * w64 * (2 * rstd_rel[:, None] + 4 * U) + U * b64
           + U * (np.abs(n) * w64 + b64))
    got = y.astype(np.float64)
    bound = HALF_STEP[dtype] * np.abs(want_y) + 2 * err + TINY[dtype]
    assert (np.abs(got - want_y) <= bound).all(), float((np.abs(got - want_y) / bound).max())


def check_backward(dtype, param, dy, x, w, mean, rstd, dx, dw, db) -> None:
    rows, cols = x.shape
    d = depth(cols)
    want_dx, want_dw, want_db, n, a = reference_backward(dy, x, w, mean, rstd)
    r = rstd.astype(np.float64)[:, None]
    abs_a, abs_n = np.abs(a), np.abs(n)
    sum_a, sum_an = abs_a.mean(axis=1, keepdims=True), (abs_a * abs_n).mean(axis=1, keepdims=True)
    # n is off by 2 u relative; the two means by d u; each of the five operations of dx adds u
    err = r * ((d + 8) * U * (sum_a + abs_n * sum_an) + 8 * U * abs_a)
    bound = HALF_STEP[dtype] * np.abs(want_dx) + 2 * err + TINY[dtype]
    got = dx.astype(np.float64)
    assert (np.abs(got - want_dx) <= bound).all(), float((np.abs(got - want_dx) / bound).max())
    # Sums over rows: at most rows / 100 of them in one chain (a CTA's rows), then the chains of the partials.
    chain = 2.0 * (rows / 100 + 64)
    dy64 = np.abs(dy.astype(np.float64))
    for got, want, size in ((dw, want_dw, (dy64 * abs_n).sum(axis=0)), (db, want_db, dy64.sum(axis=0))):
        if got is None:
            continue
        bound = HALF_STEP[param] * np.abs(want) + (chain + 4) * U * size + TINY[param]
        assert (np.abs(got.astype(np.float64) - want) <= bound).all()


def run_forward(ctx, x, w, b, ld_pad: int = 0, in_place: bool = False):
    rows, cols = x.shape
    dx_ = make(ctx, x, cols + ld_pad)
    dw_, db_ = make(ctx, w), make(ctx, b)
    dy_ = dx_ if in_place else empty(ctx, x.shape, x.dtype, cols + ld_pad)
    mean, rstd = empty(ctx, (rows,), np.float32), empty(ctx, (rows,), np.float32)
    ctx.layer_norm(dx_, dy_, weight=dw_, bias=db_, eps=EPS, mean=mean, rstd=rstd)
    ctx.synchronize()
    return dy_.to_numpy(), mean.to_numpy(), rstd.to_numpy()


def run_backward(ctx, dy, x, w, mean, rstd, ld_pad: int = 0, in_place: str = ""):
    rows, cols = x.shape
    bx, bdy = make(ctx, x, cols + ld_pad), make(ctx, dy, cols + ld_pad)
    bw, bm, br = make(ctx, w), make(ctx, mean), make(ctx, rstd)
    bdx = {"x": bx, "dy": bdy}.get(in_place) or empty(ctx, x.shape, x.dtype, cols + ld_pad)
    dw, db = empty(ctx, (cols,), w.dtype), empty(ctx, (cols,), w.dtype)
    ctx.layer_norm_backward(bdy, bx, bdx, mean=bm, rstd=br, weight=bw, dweight=dw, dbias=db)
    ctx.synchronize()
    return bdx.to_numpy(), dw.to_numpy(), db.to_numpy()


SHAPES = [(1, 1), (1, 8), (3, 5), (9, 31), (17, 64), (33, 257), (5, 512), (7, 513), (300, 1000), (2, 2049), (150, 4096),
          (5, 8191), (3, 8200), (4, 16384), (2, 33000), (1, 70001)]


@pytest.mark.parametrize("dtype, param", [("float32", "float32"), ("float16", "float16"), ("bfloat16", "bfloat16"),
                                          ("float16", "float32"), ("bfloat16", "float32")])
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_forward_and_backward(rows, cols, dtype, param, gpu_ctx) -> None:
    x, dy, w, b = inputs(rows, cols, dtype, param, 1)
    y, mean, rstd = run_forward(gpu_ctx, x, w, b)
    check_forward(dtype, x, w, b, y, mean, rstd)
    dx, dw, db = run_backward(gpu_ctx, dy, x, w, mean, rstd)
    check_backward(dtype, param, dy, x, w, mean, rstd, dx, dw, db)


@pytest.mark.parametrize("rows, cols, pad", [(40, 96, 8), (40, 96, 3), (11, 1001, 7), (6, 9000, 8), (6, 9001, 2)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_pitches_and_in_place(rows, cols, pad, dtype, gpu_ctx) -> None:
    x, dy, w, b = inputs(rows, cols, dtype, dtype, 2)
    plain = run_forward(gpu_ctx, x, w, b, pad)
    check_forward(dtype, x, w, b, *plain)
    placed = run_forward(gpu_ctx, x, w, b, pad, in_place=True)
    for p, q in zip(plain, placed):
        assert np.array_equal(p, q)
    grads = run_backward(gpu_ctx, dy, x, w, plain[1], plain[2], pad)
    check_backward(dtype, dtype, dy, x, w, plain[1], plain[2], *grads)
    for which in ("x", "dy"):
        for p, q in zip(grads, run_backward(gpu_ctx, dy, x, w, plain[1], plain[2], pad, in_place=which)):
            assert np.array_equal(p, q)


def test_rows_without_weight_bias_or_statistics(gpu_ctx) -> None:
    x, dy, _, _ = inputs(20, 300, "float32", "float32", 3)
    ones, zeros = np.ones(300, np.float32), np.zeros(300, np.float32)
    want = run_forward(gpu_ctx, x, ones, zeros)
    bx, by = make(gpu_ctx, x), empty(gpu_ctx, x.shape, x.dtype)
    gpu_ctx.layer_norm(bx, by, eps=EPS)
    gpu_ctx.synchronize()
    assert np.array_equal(by.to_numpy(), want[0])
    grads = run_backward(gpu_ctx, dy, x, ones, want[1], want[2])
    bdy, bdx = make(gpu_ctx, dy), empty(gpu_ctx, x.shape, x.dtype)
    m, r = make(gpu_ctx, want[1]), make(gpu_ctx, want[2])
    gpu_ctx.layer_norm_backward(bdy, bx, bdx, mean=m, rstd=r)
    gpu_ctx.synchronize()
    assert np.array_equal(bdx.to_numpy(), grads[0])
    only = empty(gpu_ctx, (300,), np.float32)
    gpu_ctx.layer_norm_backward(bdy, bx, bdx, mean=m, rstd=r, dbias=only)
    gpu_ctx.synchronize()
    assert np.array_equal(only.to_numpy(), grads[2])


def test_constant_rows_large_means_and_non_finite_values(gpu_ctx) -> None:
    x, dy, w, b = inputs(6, 1024, "float32", "float32", 4)
    x[0] = 3.0                                        # no variance: eps alone
    x[1] = 1000.0 + x[1]                              # a mean far above the spread
    x[2] *= 1e-12
    x[3, 7] = np.nan
    x[4, 9] = np.inf
    y, mean, rstd = run_forward(gpu_ctx, x, w, b)
    good = [0, 1, 2, 5]
    check_forward("float32", x[good], w, b, y[good], mean[good], rstd[good])
    assert np.isnan(y[3]).all() and np.isnan(y[4]).any()   # a row's trouble stays in its row


def test_many_rows_repeat_bit_for_bit(gpu_ctx) -> None:
    x, dy, w, b = inputs(5000, 256, "bfloat16", "float32", 5)
    first = run_forward(gpu_ctx, x, w, b)
    check_forward("bfloat16", x, w, b, *first)
    one = run_backward(gpu_ctx, dy, x, w, first[1], first[2])
    check_backward("bfloat16", "float32", dy, x, w, first[1], first[2], *one)
    for p, q in zip(one, run_backward(gpu_ctx, dy, x, w, first[1], first[2])):
        assert np.array_equal(p, q)


@pytest.mark.parametrize("dtype, param", [("bfloat16", "bfloat16"), ("float32", "float32"), ("float16", "float32")])
@pytest.mark.parametrize("rows, cols, pad", [(700, 300, 0), (601, 257, 0), (1500, 513, 3), (650, 1000, 0), (593, 2048, 8),
                                             (600, 2049, 0), (640, 4096, 0), (600, 5001, 2), (595, 8200, 0), (593, 16383, 0)])
def test_many_rows(rows, cols, pad, dtype, param, gpu_ctx) -> None:
    """Enough rows that every CTA walks several: rows on 16-byte boundaries and at every place between them."""
    x, dy, w, b = inputs(rows, cols, dtype, param, 8)
    y, mean, rstd = run_forward(gpu_ctx, x, w, b, pad)
    check_forward(dtype, x, w, b, y, mean, rstd)
    grads = run_backward(gpu_ctx, dy, x, w, mean, rstd, pad)
    check_backward(dtype, param, dy, x, w, mean, rstd, *grads)
    for p, q in zip(grads, run_backward(gpu_ctx, dy, x, w, mean, rstd, pad, in_place="dy")):
        assert np.array_equal(p, q)


@pytest.mark.parametrize("rows, cols, pad", [(1200, 1000, 0), (1200, 1001, 0), (2100, 1001, 4), (700, 3001, 0)])
def test_many_rows_without_weight_bias_or_statistics(rows, cols, pad, gpu_ctx) -> None:
    """Also with y's rows at other places than x's (pad)."""
    x, dy, w, b = inputs(rows, cols, "float16", "float32", 10)
    one, zero = np.ones(cols, np.float32), np.zeros(cols, np.float32)
    bx, by = make(gpu_ctx, x), empty(gpu_ctx, x.shape, x.dtype, cols + pad)
    gpu_ctx.layer_norm(bx, by, eps=EPS)
    bm, br = empty(gpu_ctx, (rows,), np.float32), empty(gpu_ctx, (rows,), np.float32)
    gpu_ctx.layer_norm(bx, empty(gpu_ctx, x.shape, x.dtype), mean=bm, rstd=br, eps=EPS)
    bdy, bdx = make(gpu_ctx, dy), empty(gpu_ctx, x.shape, x.dtype, cols + pad)
    gpu_ctx.layer_norm_backward(bdy, bx, bdx, mean=bm, rstd=br)
    gpu_ctx.synchronize()
    mean, rstd = bm.to_numpy(), br.to_numpy()
    check_forward("float16", x, one, zero, by.to_numpy(), mean, rstd)
    check_backward("float16", "float32", dy, x, one, mean, rstd, bdx.to_numpy(), None, None)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_window_of_a_larger_matrix(dtype, gpu_ctx) -> None:
    """Rows that start inside a 16-byte piece, in a buffer whose other columns are NaN and stay as they are."""
    rows, cols, left, ld = 700, 1000, 3, 1013
    x, dy, w, b = inputs(rows, cols, dtype, "float32", 9)
    t = np_dtype(dtype)

    def window(values):
        host = np.full((rows, ld), np.nan, t)
        if values is not None:
            host[:, left:left + cols] = values
        buf = make(gpu_ctx, host)
        return buf, buf.window(0, rows, left, left + cols)

    (bx, vx), (by, vy), (bd, vd), (bg, vg) = window(x), window(None), window(dy), window(None)
    bw, bb = make(gpu_ctx, w), make(gpu_ctx, b)
    mean, rstd = empty(gpu_ctx, (rows,), np.float32), empty(gpu_ctx, (rows,), np.float32)
    dw, db = empty(gpu_ctx, (cols,), np.float32), empty(gpu_ctx, (cols,), np.float32)
    gpu_ctx.layer_norm(vx, vy, weight=bw, bias=bb, eps=EPS, mean=mean, rstd=rstd)
    gpu_ctx.layer_norm_backward(vd, vx, vg, mean=mean, rstd=rstd, weight=bw, dweight=dw, dbias=db)
    gpu_ctx.synchronize()
    y, dx = by.to_numpy(), bg.to_numpy()
    check_forward(dtype, x, w, b, y[:, left:left + cols], mean.to_numpy(), rstd.to_numpy())
    check_backward(dtype, "float32", dy, x, w, mean.to_numpy(), rstd.to_numpy(), dx[:, left:left + cols], dw.to_numpy(),
                   db.to_numpy())
    for out in (y, dx):
        assert np.isnan(out[:, :left].astype(np.float32)).all() and np.isnan(out[:, left + cols:].astype(np.float32)).all()


def test_empty_problems(gpu_ctx) -> None:
    w = np.ones(8, np.float32)
    bw, dw = make(gpu_ctx, w), empty(gpu_ctx, (8,), np.float32)
    none = cuda.DeviceBuffer(gpu_ctx, (0, 8), np.float32)
    stats = cuda.DeviceBuffer(gpu_ctx, (0,), np.float32)
    gpu_ctx.layer_norm(none, none, weight=bw)
    gpu_ctx.layer_norm_backward(none, none, none, mean=stats, rstd=stats, weight=bw, dweight=dw)
    gpu_ctx.synchronize()
    assert np.array_equal(dw.to_numpy(), np.zeros(8, np.float32))
    thin = cuda.DeviceBuffer(gpu_ctx, (4, 0), np.float32)
    gpu_ctx.layer_norm(thin, thin)
    gpu_ctx.synchronize()


@pytest.mark.parametrize("rows, cols", [(6, 40), (5, 3000)])
def test_gradients_against_differences(rows, cols, gpu_ctx) -> None:
    """<dx, v> against (f(x + t v) - f(x - t v)) / 2 t of the formula in 64 bits, f = sum(y dy); the same for
    weight and bias. The quotient's own error is t^2, of second order in t = 1e-4."""
    x, dy, w, b = inputs(rows, cols, "float32", "float32", 6)
    _, mean, rstd = run_forward(gpu_ctx, x, w, b)
    dx, dw, db = run_backward(gpu_ctx, dy, x, w, mean, rstd)
    rng = np.random.default_rng(7)
    t = 1e-4

    def f(x_, w_, b_):
        return float((reference(x_, w_, b_)[0] * dy.astype(np.float64)).sum())

    for which, grad in ((0, dx), (1, dw), (2, db)):
        base = [v.astype(np.float64) for v in (x, w, b)]
        v = rng.standard_normal(base[which].shape)
        up, down = list(base), list(base)
        up[which], down[which] = base[which] + t * v, base[which] - t * v
        slope = (f(*up) - f(*down)) / (2 * t)
        got = float((grad.astype(np.float64) * v).sum())
        assert abs(got - slope) <= 1e-5 * float(np.abs(grad.astype(np.float64) * v).sum()) + 1e-6


def test_refusals_reach_python(gpu_ctx) -> None:
    a, b = empty(gpu_ctx, (4, 8), np.float32), empty(gpu_ctx, (4, 9), np.float32)
    half = empty(gpu_ctx, (8,), np.float16)
    with pytest.raises(ValueError, match="one shape and type"):
        gpu_ctx.layer_norm(a, b)
    with pytest.raises(ValueError, match="weight must be a vector of 8 elements"):
        gpu_ctx.layer_norm(a, a, weight=empty(gpu_ctx, (9,), np.float32))
    with pytest.raises(DeviceError, match="param_dtype"):
        gpu_ctx.layer_norm(a, a, weight=half)
    with pytest.raises(ValueError, match="of one type"):
        gpu_ctx.layer_norm(a, a, weight=half, bias=empty(gpu_ctx, (8,), np.float32))
    with pytest.raises(DeviceError, match="partially overlap"):
        gpu_ctx.layer_norm(a.window(0, 3, 0, 8), a.window(1, 4, 0, 8))
    ints = empty(gpu_ctx, (4, 8), np.int32)
    with pytest.raises(ValueError):
        gpu_ctx.layer_norm(ints, ints)


def test_rings_of_different_sizes_from_several_contexts_at_once() -> None:
    """The same kernels, launched by threads with a context each on rows of different widths, that is with rings of
    different sizes: no launch changes what another may ask for. (Through the C ABI with the arguments made once,
    for calls close enough together; waiting now and then, since launches that wait for room in the queue are not.)"""
    lib = cuda.library()
    programs, errors = [], []
    for rows, cols in ((148, 16384), (300, 8200)) * 2:  # 4 MiB and more: through the ring
        ctx = cuda.Context(0)
        x, dy, w, b = inputs(rows, cols, "bfloat16", "bfloat16", 41)
        bx, bdy, bw, bb = (make(ctx, v) for v in (x, dy, w, b))
        by, bdx = empty(ctx, x.shape, x.dtype), empty(ctx, x.shape, x.dtype)
        mean, rstd = empty(ctx, (rows,), np.float32), empty(ctx, (rows,), np.float32)
        dw, db = empty(ctx, (cols,), w.dtype), empty(ctx, (cols,), w.dtype)
        outputs = (by, mean, rstd, bdx, dw, db)
        ctx.layer_norm(bx, by, weight=bw, bias=bb, eps=EPS, mean=mean, rstd=rstd)
        ctx.layer_norm_backward(bdy, bx, bdx, mean=mean, rstd=rstd, weight=bw, dweight=dw, dbias=db)
        ctx.synchronize()
        alone = [out.to_numpy() for out in outputs]
        check_forward("bfloat16", x, w, b, *alone[:3])
        check_backward("bfloat16", "bfloat16", dy, x, w, alone[1], alone[2], *alone[3:])
        args = (cuda._LayerNormArgs(rows, cols, cuda.C_BF16, cuda.C_BF16, bx.ptr, cols, bw.ptr, bb.ptr, by.ptr, cols, mean.ptr,
                                    rstd.ptr, EPS),
                cuda._LayerNormBackwardArgs(rows, cols, cuda.C_BF16, cuda.C_BF16, bdy.ptr, cols, bx.ptr, cols, bw.ptr, mean.ptr,
                                            rstd.ptr, bdx.ptr, cols, dw.ptr, db.ptr))
        programs.append((ctx, args, outputs, alone, (bx, bdy, bw, bb)))

    def work(ctx, args):
        forward, backward = (ctypes.byref(a) for a in args)
        failed = 0
        for _ in range(1500):
            for _ in range(4):
                failed += lib.hcCudaLayerNorm(ctx._handle, forward) != 0
                failed += lib.hcCudaLayerNormBackward(ctx._handle, backward) != 0
            ctx.synchronize()
        errors.append(failed)

    threads = [threading.Thread(target=work, args=program[:2]) for program in programs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert errors == [0] * len(programs)
    for _, _, outputs, alone, _ in programs:
        for out, before in zip(outputs, alone):
            assert np.array_equal(out.to_numpy(), before)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cols", [1, 8, 64, 512, 2048])
def test_constant_rows_of_huge_values(cols, dtype, gpu_ctx) -> None:
    """Rows of one value, 2^110, whose mean is exact (cols is a power of two): n is 0, although mean * rstd, with
    rstd = 2^20 for eps = 2^-40, is beyond float32. Lanes and threads that hold nothing of the row add nothing."""
    rng = np.random.default_rng(cols)
    t, eps = np_dtype(dtype), 2.0**-40
    x = np.full((5, cols), 2.0**110).astype(t)
    dy = rng.standard_normal((5, cols)).astype(t)
    w, b = rng.standard_normal(cols).astype(np.float32), rng.standard_normal(cols).astype(np.float32)
    bx, bdy, bw, bb = (make(gpu_ctx, v) for v in (x, dy, w, b))
    y, dx = empty(gpu_ctx, x.shape, t), empty(gpu_ctx, x.shape, t)
    mean, rstd = empty(gpu_ctx, (5,), np.float32), empty(gpu_ctx, (5,), np.float32)
    dw, db = empty(gpu_ctx, (cols,), np.float32), empty(gpu_ctx, (cols,), np.float32)
    gpu_ctx.layer_norm(bx, y, weight=bw, bias=bb, eps=eps, mean=mean, rstd=rstd)
    gpu_ctx.layer_norm_backward(bdy, bx, dx, mean=mean, rstd=rstd, weight=bw, dweight=dw, dbias=db)
    gpu_ctx.synchronize()
    m, r = mean.to_numpy(), rstd.to_numpy()
    assert (m == 2.0**110).all() and (np.abs(r - 2.0**20) <= 8 * U * 2.0**20).all()
    assert (np.abs(y.to_numpy().astype(np.float64) - b.astype(np.float64)) <= HALF_STEP[dtype] * np.abs(b)).all()
    check_backward(dtype, "float32", dy, x, w, m, r, dx.to_numpy(), dw.to_numpy(), db.to_numpy())


@pytest.mark.parametrize("dtype, cols", [("bfloat16", 4096), ("float16", 1032), ("float32", 2048), ("bfloat16", 16384)])
def test_a_row_gives_the_same_bits_wherever_it_stands(dtype, cols, gpu_ctx) -> None:
    """The same rows many times over: rings that every CTA refills again and again, each row's y and dx as the first
    time, and so in every run. (Rows on 16-byte boundaries: a row's sums do not depend on where it lies.)"""
    block, copies = 96, (1 << 25) // (96 * cols)
    x, dy, w, b = inputs(block, cols, dtype, "float32", 61)
    t = np_dtype(dtype)
    big = [empty(gpu_ctx, (block * copies, cols), t) for _ in range(4)]
    for buf, v in zip(big, (x, dy)):
        for i in range(copies):
            buf.window(i * block, (i + 1) * block, 0, cols).copy_from_host(v)
    bx, bdy, by, bdx = big
    bw, bb = make(gpu_ctx, w), make(gpu_ctx, b)
    mean, rstd = (empty(gpu_ctx, (block * copies,), np.float32) for _ in range(2))
    dw, db = (empty(gpu_ctx, (cols,), np.float32) for _ in range(2))
    sums = None
    for _ in range(3):
        for buf in (by, bdx, mean, rstd, dw, db):
            buf.fill_bytes(0xFF)
        gpu_ctx.layer_norm(bx, by, weight=bw, bias=bb, eps=EPS, mean=mean, rstd=rstd)
        gpu_ctx.layer_norm_backward(bdy, bx, bdx, mean=mean, rstd=rstd, weight=bw, dweight=dw, dbias=db)
        gpu_ctx.synchronize()
        y, dx = (buf.to_numpy().reshape(copies, block, cols) for buf in (by, bdx))
        assert (y == y[0]).all() and (dx == dx[0]).all()
        again = dw.to_numpy(), db.to_numpy()
        assert sums is None or all(np.array_equal(p, q) for p, q in zip(sums, again))
        sums = again
    m, r = mean.to_numpy()[:block], rstd.to_numpy()[:block]
    check_forward(dtype, x, w, b, y[0], m, r)
    check_backward(dtype, "float32", dy, x, w, m, r, dx[0], None, None)


@pytest.mark.parametrize("rows, cols, pad", [(1200, 4096, 0), (1200, 4095, 0), (700, 8200, 0), (900, 5001, 3)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_many_rows_in_place(dtype, rows, cols, pad, gpu_ctx) -> None:
    """y written over x, and dx over x and over dy, where rows are read some rows ahead."""
    x, dy, w, b = inputs(rows, cols, dtype, "float32", 62)
    apart = run_forward(gpu_ctx, x, w, b, pad)
    for p, q in zip(apart, run_forward(gpu_ctx, x, w, b, pad, in_place=True)):
        assert np.array_equal(p, q)
    grads = run_backward(gpu_ctx, dy, x, w, apart[1], apart[2], pad)
    for which in ("x", "dy"):
        for p, q in zip(grads, run_backward(gpu_ctx, dy, x, w, apart[1], apart[2], pad, in_place=which)):
            assert np.array_equal(p, q)


@pytest.mark.parametrize("rows, cols", [(5, 64), (300, 1000), (700, 4096), (700, 4095)])
@pytest.mark.parametrize("param", ["bfloat16", "float32"])
def test_vectors_at_any_address(param, rows, cols, gpu_ctx) -> None:
    """Weight, bias, their gradients and the statistics at addresses that are multiples of their element alone."""
    x, dy, w, b = inputs(rows, cols, "bfloat16", param, 71)
    keep = []

    def odd(values, length, dtype):
        dtype = np.dtype(dtype)
        raw = empty(gpu_ctx, (length + 2,), dtype)
        keep.append(raw)
        if values is not None:
            raw.copy_from_host(np.concatenate([np.full(1, np.nan, dtype), values, np.full(1, np.nan, dtype)]))
        return raw, cuda.DeviceBuffer.wrap(gpu_ctx, raw.ptr + dtype.itemsize, (length,), dtype)

    (_, vw), (_, vb) = odd(w, cols, w.dtype), odd(b, cols, b.dtype)
    outs = [odd(None, rows, np.float32), odd(None, rows, np.float32), odd(None, cols, w.dtype), odd(None, cols, w.dtype)]
    (_, mean), (_, rstd), (_, dw), (_, db) = outs
    bx, bdy = make(gpu_ctx, x), make(gpu_ctx, dy)
    y, dx = empty(gpu_ctx, x.shape, x.dtype), empty(gpu_ctx, x.shape, x.dtype)
    gpu_ctx.layer_norm(bx, y, weight=vw, bias=vb, eps=EPS, mean=mean, rstd=rstd)
    gpu_ctx.layer_norm_backward(bdy, bx, dx, mean=mean, rstd=rstd, weight=vw, dweight=dw, dbias=db)
    gpu_ctx.synchronize()
    got = [raw.to_numpy() for raw, _ in outs]
    for v in got:  # nothing beside a vector is written
        assert (v[[0, -1]].view(np.uint8) == 0xFF).all()
    m, r, gw, gb = (v[1:-1] for v in got)
    check_forward("bfloat16", x, w, b, y.to_numpy(), m, r)
    check_backward("bfloat16", param, dy, x, w, m, r, dx.to_numpy(), gw, gb)
