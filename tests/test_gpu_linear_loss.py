"""The linear cross entropy and its gradients on a B200 against the formula in 64 bits.

Tolerances. u = 2^-24. A product of two 16-bit values is exact in float32; the tensor cores add 16 of
them and the accumulator at a time, cutting at most 2^-22 of what they add: a logit is off by at most
E = (width / 16 + 8) 2^-22 sum|h w|. An exponential adds 2^-21 relative (its argument's rounding and the
instruction's own error), the sum over the vocabulary of positive terms (vocab / 256 + 64) u relative, the
logarithm and its neighbours 8 u (1 + |lse|). Gradients: an entry of g carries the rounding to its type, h, and
P = E + 2^-20 + 8 u (1 + |lse|) relative on its exponential; the products add what they add to the logits and
one rounding of the result.
"""

from __future__ import annotations

import numpy as np
import pytest

from conftest import np_dtype
from hc import cuda
from hc.errors import DeviceError

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF_STEP = {"float16": 2.0**-11, "bfloat16": 2.0**-8}
TINY = {"float16": 2.0**-25, "bfloat16": 2.0**-133}
IGNORE = -100


def make(ctx, array: np.ndarray, ld: int | None = None) -> cuda.DeviceBuffer:
    buf = empty(ctx, array.shape, array.dtype, ld)
    buf.copy_from_host(array)
    return buf


def empty(ctx, shape, dtype, ld: int | None = None) -> cuda.DeviceBuffer:
    buf = cuda.DeviceBuffer(ctx, shape, dtype, ld=ld)
    if buf.nbytes:
        buf.fill_bytes(0xFF)
    return buf


def inputs(rows, vocab, width, dtype, seed=1, sure=3.0):
    rng = np.random.default_rng([rows, vocab, width, seed])
    t = np_dtype(dtype)
    w = (rng.standard_normal((vocab, width)) / np.sqrt(width)).astype(t)
    targets = rng.integers(0, vocab, rows)
    h = (rng.standard_normal((rows, width)) + sure * rng.random((rows, 1)) * w[targets].astype(np.float64)).astype(t)
    targets[rng.random(rows) < 0.1] = IGNORE
    dloss = (rng.standard_normal(rows) / rows).astype(np.float32)
    return h, w, targets.astype(np.int64), dloss


class Exact:
    def __init__(self, h, w, targets, dloss):
        h, w = h.astype(np.float64), w.astype(np.float64)
        rows, vocab = h.shape[0], w.shape[0]
        width = h.shape[1]
        logits = h @ w.T
        size = np.abs(h) @ np.abs(w).T
        top = logits.max(axis=1)
        p = np.exp(logits - top[:, None])
        self.lse = np.log(p.sum(axis=1)) + top
        self.counts = (targets != IGNORE) & (targets >= 0) & (targets < vocab)
        at = np.where(self.counts, targets, 0)
        rng = np.arange(rows)
        self.loss = np.where(targets == IGNORE, 0.0, np.where(self.counts, self.lse - logits[rng, at], np.nan))
        e_logit = (width / 16 + 8) * 2.0**-22 * size
        own = 8 * U * (1 + np.abs(self.lse))
        self.lse_bound = e_logit.max(axis=1) + (vocab / 256 + 64) * U + 2.0**-21 + own
        self.loss_bound = self.lse_bound + e_logit[rng, at] + U * np.abs(np.nan_to_num(self.loss))
        p = np.exp(logits - self.lse[:, None])
        g = p.copy()
        g[rng[self.counts], at[self.counts]] -= 1.0
        scale = np.where(self.counts, dloss.astype(np.float64), 0.0)[:, None]
        self.g, self.p, self.scale = g * scale, p, scale
        self.p_rel = e_logit + (self.lse_bound + 2.0**-20 + own)[:, None]
        self.h, self.w = h, w
        self.dh, self.dw = self.g @ w, self.g.T @ h

    def bounds(self, dtype):
        # float16: g is scaled so that the largest |dloss| stands for 2^14, and keeps that many times more below
        # the type's smallest normal number (2^13 leaves a factor of two).
        step = HALF_STEP[dtype]
        floor = 2.0**-25 * np.abs(self.scale).max() * 2.0**-13 if dtype == "float16" else 0.0
        g_err = np.abs(self.g) * step + np.abs(self.scale) * self.p * self.p_rel * (1 + step) + floor
        g_err = np.where(self.scale == 0.0, 0.0, g_err)
        rows, vocab = self.g.shape
        ga = np.abs(self.g) + g_err
        dh = g_err @ np.abs(self.w) + (vocab / 16 + 64) * 2.0**-22 * (ga @ np.abs(self.w))
        dw = g_err.T @ np.abs(self.h) + (rows / 16 + 64) * 2.0**-22 * (ga.T @ np.abs(self.h))
        return (dh * (1 + step) + step * np.abs(self.dh) + TINY[dtype], dw * (1 + step) + step * np.abs(self.dw) + TINY[dtype])


def run(ctx, h, w, targets, dloss, pad_h=0, pad_w=0, want=("dh", "dw"), ignore=IGNORE):
    rows, width = h.shape
    bh, bw = make(ctx, h, width + pad_h), make(ctx, w, width + pad_w)
    bt, bd = make(ctx, targets), make(ctx, dloss)
    loss, lse = empty(ctx, (rows,), np.float32), empty(ctx, (rows,), np.float32)
    ctx.linear_cross_entropy(bh, bw, bt, loss, lse, ignore_index=ignore)
    dh = empty(ctx, h.shape, h.dtype, width + pad_h) if "dh" in want else None
    dw = empty(ctx, w.shape, w.dtype, width + pad_w) if "dw" in want else None
    ctx.linear_cross_entropy_backward(bh, bw, bt, lse, bd, dh=dh, dw=dw, ignore_index=ignore)
    ctx.synchronize()
    return (loss.to_numpy(), lse.to_numpy(), None if dh is None else dh.to_numpy(), None if dw is None else dw.to_numpy())


def check(dtype, exact, loss, lse, dh, dw) -> None:
    assert (np.abs(lse - exact.lse) <= exact.lse_bound).all()
    nan = np.isnan(exact.loss)
    assert np.array_equal(np.isnan(loss), nan)
    assert (np.abs(loss - exact.loss)[~nan] <= exact.loss_bound[~nan]).all()
    bound_h, bound_w = exact.bounds(dtype)
    if dh is not None:
        assert (np.abs(dh.astype(np.float64) - exact.dh) <= bound_h).all()
        assert (dh.astype(np.float64)[~exact.counts] == 0).all()
    if dw is not None:
        assert (np.abs(dw.astype(np.float64) - exact.dw) <= bound_w).all()


SHAPES = [(1, 1, 1), (1, 300, 64), (3, 7, 9), (31, 257, 40), (129, 1000, 128), (257, 513, 100), (300, 2051, 333),
          (64, 5000, 1000), (520, 770, 264)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows, vocab, width", SHAPES)
def test_loss_and_gradients(rows, vocab, width, dtype, gpu_ctx) -> None:
    h, w, targets, dloss = inputs(rows, vocab, width, dtype)
    check(dtype, Exact(h, w, targets, dloss), *run(gpu_ctx, h, w, targets, dloss))


@pytest.mark.parametrize("rows, vocab, width", [(1, 40000, 72), (8, 30001, 64), (53, 20000, 80), (127, 10000, 64), (385, 6000, 64)])
def test_few_rows_and_a_large_vocabulary(rows, vocab, width, gpu_ctx) -> None:
    """Several tiles per SM whose rows do not fill the tile."""
    h, w, targets, dloss = inputs(rows, vocab, width, "bfloat16", 11)
    targets[0] = vocab - 1
    check("bfloat16", Exact(h, w, targets, dloss), *run(gpu_ctx, h, w, targets, dloss))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("piece", ["256", "512", "1024"])
def test_pieces_of_the_vocabulary(piece, dtype, gpu_ctx, monkeypatch) -> None:
    h, w, targets, dloss = inputs(150, 1300, 200, dtype, 2)
    exact = Exact(h, w, targets, dloss)
    monkeypatch.setenv("HC_CUDA_LOSS_PIECE", piece)
    first = run(gpu_ctx, h, w, targets, dloss)
    check(dtype, exact, *first)
    for a, b in zip(first, run(gpu_ctx, h, w, targets, dloss)):
        assert np.array_equal(a, b)  # the same bits every time


@pytest.mark.parametrize("rows, width", [(150, 201), (33, 515)])
def test_pieces_at_odd_places(rows, width, gpu_ctx, monkeypatch) -> None:
    h, w, targets, dloss = inputs(rows, 1300, width, "float16", 12)
    monkeypatch.setenv("HC_CUDA_LOSS_PIECE", "512")
    check("float16", Exact(h, w, targets, dloss), *run(gpu_ctx, h, w, targets, dloss, 0, 0))
    check("float16", Exact(h, w, targets, dloss), *run(gpu_ctx, h, w, targets, dloss, 2, 1))


@pytest.mark.parametrize("pad_h, pad_w", [(8, 16), (1, 0), (0, 3), (5, 1)])
def test_pitches(pad_h, pad_w, gpu_ctx) -> None:
    h, w, targets, dloss = inputs(70, 600, 96, "bfloat16", 3)
    check("bfloat16", Exact(h, w, targets, dloss), *run(gpu_ctx, h, w, targets, dloss, pad_h, pad_w))


def test_one_gradient_alone_and_32_bit_targets(gpu_ctx) -> None:
    h, w, targets, dloss = inputs(90, 700, 64, "bfloat16", 4)
    both = run(gpu_ctx, h, w, targets, dloss)
    check("bfloat16", Exact(h, w, targets, dloss), *both)
    only_h = run(gpu_ctx, h, w, targets.astype(np.int32), dloss, want=("dh",))
    only_w = run(gpu_ctx, h, w, targets, dloss, want=("dw",))
    assert np.array_equal(only_h[0], both[0]) and np.array_equal(only_h[2], both[2]) and only_h[3] is None
    assert np.array_equal(only_w[3], both[3]) and only_w[2] is None


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_rows_that_do_not_count(dtype, gpu_ctx) -> None:
    """Ignored rows have loss 0, targets outside the vocabulary NaN, and neither adds to a gradient --
    whatever their dloss or their values; a batch of ignored rows alone gives zero gradients."""
    h, w, targets, dloss = inputs(40, 300, 64, dtype, 5)
    targets[:] = np.arange(40) * 7
    targets[3], targets[4], targets[5] = IGNORE, 300, -1
    h[6, 2], targets[6] = np.nan, IGNORE
    dloss[3], dloss[4] = np.nan, np.inf
    loss, lse, dh, dw = run(gpu_ctx, h, w, targets, dloss)
    clean = h.copy()
    clean[6] = 0
    exact = Exact(clean, w, targets, dloss)
    assert np.isnan(lse[6]) and loss[6] == 0 and (dh[6] == 0).all()
    lse[6] = exact.lse[6]
    keep = exact.counts
    bound_h, bound_w = exact.bounds(dtype)
    assert (np.abs(dh.astype(np.float64) - exact.dh)[keep] <= bound_h[keep]).all()
    assert (dh.astype(np.float64)[~keep] == 0).all()
    assert (np.abs(dw.astype(np.float64) - exact.dw) <= bound_w).all()  # no trace of the NaN either
    assert np.isnan(loss[4]) and np.isnan(loss[5]) and loss[3] == 0
    targets[:] = IGNORE
    loss, _, dh, dw = run(gpu_ctx, h, w, targets, dloss)
    assert (loss == 0).all() and (dh.astype(np.float64) == 0).all() and (dw.astype(np.float64) == 0).all()


def test_another_ignore_index(gpu_ctx) -> None:
    h, w, targets, dloss = inputs(40, 300, 64, "bfloat16", 6)
    targets = np.abs(targets) % 300
    targets[::3] = 17
    loss, _, dh, _ = run(gpu_ctx, h, w, targets, dloss, ignore=17)
    assert (loss[::3] == 0).all() and (dh.astype(np.float64)[::3] == 0).all() and (loss[1::3] > 0).all()


def test_large_logits_and_sure_rows(gpu_ctx) -> None:
    """Logits of several hundred: exponentials of the differences, never of the logits; and rows whose
    target has all of the probability."""
    h, w, targets, dloss = inputs(60, 900, 128, "bfloat16", 7, sure=40.0)
    h = (h.astype(np.float64) * 8).astype(h.dtype)
    check("bfloat16", Exact(h, w, targets, dloss), *run(gpu_ctx, h, w, targets, dloss))


def test_tiny_and_huge_upstream_factors_in_float16(gpu_ctx) -> None:
    for size in (1e-12, 1.0, 3e4):
        h, w, targets, dloss = inputs(50, 400, 64, "float16", 8)
        dloss = (dloss * 50 * size).astype(np.float32)
        exact = Exact(h, w, targets, dloss)
        loss, lse, dh, dw = run(gpu_ctx, h, w, targets, dloss)
        bound_h, bound_w = exact.bounds("float16")
        fits_h, fits_w = np.abs(exact.dh) < 6e4, np.abs(exact.dw) < 6e4
        assert (np.abs(dh.astype(np.float64) - exact.dh) <= bound_h)[fits_h].all()
        assert (np.abs(dw.astype(np.float64) - exact.dw) <= bound_w)[fits_w].all()


def test_no_rows(gpu_ctx) -> None:
    w = np.ones((50, 16), np.float16)
    bh, bt = cuda.DeviceBuffer(gpu_ctx, (0, 16), np.float16), cuda.DeviceBuffer(gpu_ctx, (0,), np.int64)
    bw, dw = make(gpu_ctx, w), empty(gpu_ctx, (50, 16), np.float16, 20)
    none = cuda.DeviceBuffer(gpu_ctx, (0,), np.float32)
    gpu_ctx.linear_cross_entropy(bh, bw, bt, none, none)
    gpu_ctx.linear_cross_entropy_backward(bh, bw, bt, none, none, dh=bh, dw=dw)
    gpu_ctx.synchronize()
    assert (dw.to_numpy() == 0).all()


def test_gradients_against_differences(gpu_ctx) -> None:
    """<dh, v> and <dw, v> against the differences of sum(loss dloss) of the formula in 64 bits, for
    t = 1e-4: what is left is the rounding of g (h of its type per entry) and of the gradient itself."""
    h, w, targets, dloss = inputs(30, 200, 48, "float16", 9)
    dloss = np.abs(dloss)
    _, _, dh, dw = run(gpu_ctx, h, w, targets, dloss)
    rng = np.random.default_rng(10)
    bound_h, bound_w = Exact(h, w, targets, dloss).bounds("float16")

    def f(h_, w_):
        e = Exact(h_, w_, targets, dloss)
        return float((e.loss * dloss.astype(np.float64)).sum())

    t = 1e-4
    for which, grad, bound in ((0, dh, bound_h), (1, dw, bound_w)):
        base = [h.astype(np.float64), w.astype(np.float64)]
        v = rng.standard_normal(base[which].shape)
        up, down = list(base), list(base)
        up[which], down[which] = base[which] + t * v, base[which] - t * v
        slope = (f(*up) - f(*down)) / (2 * t)
        assert abs(float((grad.astype(np.float64) * v).sum()) - slope) <= float((bound * np.abs(v)).sum()) + 1e-6


def test_refusals_reach_python(gpu_ctx) -> None:
    h, w = empty(gpu_ctx, (4, 8), np.float16), empty(gpu_ctx, (9, 8), np.float16)
    t, f = empty(gpu_ctx, (4,), np.int64), empty(gpu_ctx, (4,), np.float32)
    g = empty(gpu_ctx, (4,), np.float32)
    with pytest.raises(ValueError, match="of one type"):
        gpu_ctx.linear_cross_entropy(h, empty(gpu_ctx, (9, 7), np.float16), t, f, g)
    with pytest.raises(ValueError, match="targets must be a vector of 4 elements"):
        gpu_ctx.linear_cross_entropy(h, w, f, f, g)
    with pytest.raises(ValueError, match="loss must be a vector of 4 elements"):
        gpu_ctx.linear_cross_entropy(h, w, t, empty(gpu_ctx, (5,), np.float32), g)
    with pytest.raises(DeviceError, match="loss must not overlap lse"):
        gpu_ctx.linear_cross_entropy(h, w, t, f, f)
    with pytest.raises(ValueError, match="dw must have the shape and type of w"):
        gpu_ctx.linear_cross_entropy_backward(h, w, t, f, g, dw=h)
    with pytest.raises(ValueError, match="multiplies"):
        single = empty(gpu_ctx, (4, 8), np.float32)
        gpu_ctx.linear_cross_entropy(single, single, t, f, g)


@pytest.mark.parametrize("rows, vocab, width", [(48, 3000, 64), (300, 900, 40), (31, 700, 33)])
@pytest.mark.parametrize("piece", [None, "512"])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_rows_of_very_different_upstream_factors(dtype, piece, rows, vocab, width, gpu_ctx, monkeypatch) -> None:
    """dloss from 1e5 down to 1e-5 of it and less in one batch, flat distributions (p near 1 / vocab): every row of dh is
    as exact as if it were alone. In float16 an entry of its g is off by half a step, at least 2^-25 below the 2^14
    that stands for 1 (2^13 leaves a factor of two): nothing of another row's dloss."""
    if piece is not None:
        monkeypatch.setenv("HC_CUDA_LOSS_PIECE", piece)
    h, w, targets, _ = inputs(rows, vocab, width, dtype, 13, sure=0.0)
    h = (h.astype(np.float64) / 8).astype(h.dtype)
    w = (w.astype(np.float64) * 4).astype(w.dtype)
    dloss = (1e5 * 10.0 ** -np.linspace(0, 9, rows)).astype(np.float32) * np.where(np.arange(rows) % 3, 1, -1).astype(np.float32)
    targets[[0, rows // 2]] = IGNORE, 1
    loss, lse, dh, dw = run(gpu_ctx, h, w, targets, dloss)
    exact = Exact(h, w, targets, dloss)
    step = HALF_STEP[dtype]
    size = np.abs(exact.scale)
    floor = 2.0**-38 * size if dtype == "float16" else 0.0
    g_err = np.where(size == 0, 0.0, np.abs(exact.g) * step + size * exact.p * exact.p_rel * (1 + step) + floor)
    sums = (np.abs(exact.g) + g_err) @ np.abs(exact.w)
    bound = (g_err @ np.abs(exact.w) + (vocab / 16 + 64) * 2.0**-22 * sums) * (1 + step) + step * np.abs(exact.dh) + TINY[dtype]
    # (What lies beyond float16's 65504 is infinite there; below 6e4 the bound cannot reach it.)
    fits_h, fits_w = np.abs(exact.dh) < 6e4, np.abs(exact.dw) < 6e4
    assert (np.abs(dh.astype(np.float64) - exact.dh) <= bound)[fits_h].all()
    # dw is a sum over the rows: exact next to the largest dloss.
    assert (np.abs(dw.astype(np.float64) - exact.dw) <= exact.bounds(dtype)[1])[fits_w].all()
    if dtype == "float16":
        assert np.array_equal(dh[np.abs(exact.dh) > 7e4], np.copysign(np.inf, exact.dh[np.abs(exact.dh) > 7e4]))


@pytest.mark.parametrize("width", [500, 1024, 1025, 2049, 4096, 9000, 20000])
def test_long_sums_of_one_sign(width, gpu_ctx) -> None:
    """Products that are all positive, so that whatever an addition cuts off is cut off every time. The tensor cores
    add 1024 of the width (64 additions, and the 8 of the other tests' bound), these sums are added with rounding."""
    rows, vocab = 64, 600
    rng = np.random.default_rng(width)
    h = (0.5 + 0.5 * rng.random((rows, width))).astype(np.float16)
    w = ((0.5 + 0.5 * rng.random((vocab, width))) * (20 / (0.5625 * width))).astype(np.float16)
    targets = rng.integers(0, vocab, rows)
    dloss = (rng.standard_normal(rows) / rows).astype(np.float32)
    loss, lse, dh, dw = run(gpu_ctx, h, w, targets, dloss)
    exact = Exact(h, w, targets, dloss)
    size = np.abs(exact.h) @ np.abs(exact.w).T
    e_logit = (min(width, 1024) / 16 + 8 + width / 4096) * 2.0**-22 * size
    own = 8 * U * (1 + np.abs(exact.lse))
    exact.lse_bound = e_logit.max(axis=1) + (vocab / 256 + 64) * U + 2.0**-21 + own
    exact.loss_bound = exact.lse_bound + e_logit[np.arange(rows), targets] + U * np.abs(exact.loss)
    exact.p_rel = e_logit + (exact.lse_bound + 2.0**-20 + own)[:, None]
    check("float16", exact, loss, lse, dh, dw)


@pytest.mark.parametrize("rows, vocab, width", [(70, 600, 96), (300, 2051, 129), (5, 300, 64)])
@pytest.mark.parametrize("left", [1, 4, 8])
def test_windows_of_larger_matrices(left, rows, vocab, width, gpu_ctx) -> None:
    """h, w and both gradients inside rows of larger buffers, whose other columns stay as they are."""
    for dtype in ("bfloat16", "float16"):
        h, w, targets, dloss = inputs(rows, vocab, width, dtype, 14)

        def window(values, fill=0x5A):
            host = np.zeros((values.shape[0], left + width + 3), values.dtype)
            host.view(np.uint8)[:] = fill
            host[:, left:left + width] = values
            buf = make(gpu_ctx, host)
            return buf, buf.window(0, values.shape[0], left, left + width)

        (bh, vh), (bw, vw), (gh, dh), (gw, dw) = window(h), window(w), window(h), window(w)
        bt, bd = make(gpu_ctx, targets), make(gpu_ctx, dloss)
        loss, lse = empty(gpu_ctx, (rows,), np.float32), empty(gpu_ctx, (rows,), np.float32)
        gpu_ctx.linear_cross_entropy(vh, vw, bt, loss, lse)
        gpu_ctx.linear_cross_entropy_backward(vh, vw, bt, lse, bd, dh=dh, dw=dw)
        gpu_ctx.synchronize()
        got = [buf.to_numpy() for buf in (gh, gw)]
        assert bh.ptr and bw.ptr  # (a window does not keep the buffer it lies in)
        check(dtype, Exact(h, w, targets, dloss), loss.to_numpy(), lse.to_numpy(),
              *(np.ascontiguousarray(v[:, left:left + width]) for v in got))
        for v in got:
            for beside in (v[:, :left], v[:, left + width:]):
                assert (np.ascontiguousarray(beside).view(np.uint8) == 0x5A).all()


@pytest.mark.parametrize("rows, vocab, width", [(1, 37, 7), (70, 600, 95), (300, 2051, 130), (700, 300, 1001), (640, 2500, 516),
                                               (2500, 900, 1030)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_widths_that_end_inside_a_piece(dtype, rows, vocab, width, gpu_ctx) -> None:
    """Rows that start on 16-byte boundaries and end inside a 16-byte piece: the elements behind them stay."""
    h, w, targets, dloss = inputs(rows, vocab, width, dtype, 15)
    ld = (width + 7) // 8 * 8
    bh, bw, bt, bd = make(gpu_ctx, h, ld), make(gpu_ctx, w, ld), make(gpu_ctx, targets), make(gpu_ctx, dloss)
    gh, gw = empty(gpu_ctx, (rows, ld), h.dtype), empty(gpu_ctx, (vocab, ld), h.dtype)
    loss, lse = empty(gpu_ctx, (rows,), np.float32), empty(gpu_ctx, (rows,), np.float32)
    gpu_ctx.linear_cross_entropy(bh, bw, bt, loss, lse)
    gpu_ctx.linear_cross_entropy_backward(bh, bw, bt, lse, bd, dh=gh.window(0, rows, 0, width), dw=gw.window(0, vocab, 0, width))
    gpu_ctx.synchronize()
    dh, dw = gh.to_numpy(), gw.to_numpy()
    for out in (dh, dw):
        assert (np.ascontiguousarray(out[:, width:]).view(np.uint8) == 0xFF).all()
    check(dtype, Exact(h, w, targets, dloss), loss.to_numpy(), lse.to_numpy(), np.ascontiguousarray(dh[:, :width]),
          np.ascontiguousarray(dw[:, :width]))
