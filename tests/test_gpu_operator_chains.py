"""The operators of a language model one after another on a B200, as a program has them: nothing waits between
the calls, each reads what the one before wrote. Every link is then checked against its formula in 64 bits on the
very inputs it had, with the tolerances of its own tests."""

from __future__ import annotations

import threading

import numpy as np
import pytest

import test_gpu_gemm_w4 as w4
import test_gpu_linear_loss as loss
import test_gpu_norm as norm
from conftest import np_dtype
from hc import cuda
from hc.errors import DeviceError

pytestmark = pytest.mark.gpu


class TrainingStep:
    """Layer norm, the loss of the layer behind it, and the gradients of both."""

    def __init__(self, ctx, rows, vocab, width, dtype):
        self.ctx, self.dtype = ctx, dtype
        self.x, _, self.weight, self.bias = norm.inputs(rows, width, dtype, "float32", 21)
        _, self.w, self.targets, self.dloss = loss.inputs(rows, vocab, width, dtype, 22)
        t = np_dtype(dtype)
        self.bx, self.bw, self.bt = (norm.make(ctx, v) for v in (self.x, self.w, self.targets))
        self.bweight, self.bbias, self.bdloss = (norm.make(ctx, v) for v in (self.weight, self.bias, self.dloss))
        self.mean, self.rstd, self.loss, self.lse = (norm.empty(ctx, (rows,), np.float32) for _ in range(4))
        self.h, self.dh, self.dx = (norm.empty(ctx, (rows, width), t) for _ in range(3))
        self.dw = norm.empty(ctx, (vocab, width), t)
        self.dweight, self.dbias = (norm.empty(ctx, (width,), np.float32) for _ in range(2))

    def enqueue(self):
        c = self.ctx
        c.layer_norm(self.bx, self.h, weight=self.bweight, bias=self.bbias, eps=norm.EPS, mean=self.mean, rstd=self.rstd)
        c.linear_cross_entropy(self.h, self.bw, self.bt, self.loss, self.lse)
        c.linear_cross_entropy_backward(self.h, self.bw, self.bt, self.lse, self.bdloss, dh=self.dh, dw=self.dw)
        c.layer_norm_backward(self.dh, self.bx, self.dx, mean=self.mean, rstd=self.rstd, weight=self.bweight,
                              dweight=self.dweight, dbias=self.dbias)

    def results(self):
        names = ("h", "mean", "rstd", "loss", "lse", "dh", "dw", "dx", "dweight", "dbias")
        return {name: getattr(self, name).to_numpy() for name in names}

    def check(self, r):
        norm.check_forward(self.dtype, self.x, self.weight, self.bias, r["h"], r["mean"], r["rstd"])
        exact = loss.Exact(r["h"], self.w, self.targets, self.dloss)
        loss.check(self.dtype, exact, r["loss"], r["lse"], r["dh"], r["dw"])
        norm.check_backward(self.dtype, "float32", r["dh"], self.x, self.weight, r["mean"], r["rstd"], r["dx"],
                            r["dweight"], r["dbias"])


class Token:
    """The norm of a few tokens and two products with 4-bit weights behind it, the second of the first's result."""

    def __init__(self, ctx, m, width, inner, group, dtype):
        self.ctx, self.dtype, self.group = ctx, dtype, group
        self.x, _, self.weight, self.bias = norm.inputs(m, width, dtype, "float32", 31)
        _, self.up, self.up_scales, self.up_zeros = w4.inputs(m, inner, width, group, dtype, True, 32)
        _, self.down, self.down_scales, _ = w4.inputs(m, width, inner, group, dtype, False, 33)
        t = np_dtype(dtype)
        self.bx, self.bweight, self.bbias = (norm.make(ctx, v) for v in (self.x, self.weight, self.bias))
        self.bup = [norm.make(ctx, v) for v in (self.up, self.up_scales, self.up_zeros)]
        self.bdown = [norm.make(ctx, v) for v in (self.down, self.down_scales)]
        self.y, self.a = norm.empty(ctx, (m, width), t), norm.empty(ctx, (m, inner), t)
        self.c = norm.empty(ctx, (m, width), np.float32)
        self.mean, self.rstd = norm.empty(ctx, (m,), np.float32), norm.empty(ctx, (m,), np.float32)

    def enqueue(self):
        self.ctx.layer_norm(self.bx, self.y, weight=self.bweight, bias=self.bbias, eps=norm.EPS, mean=self.mean, rstd=self.rstd)
        self.ctx.gemm_w4(self.y, self.bup[0], self.bup[1], self.a, group=self.group, zeros=self.bup[2])
        self.ctx.gemm_w4(self.a, self.bdown[0], self.bdown[1], self.c, group=self.group)

    def results(self):
        return {name: getattr(self, name).to_numpy() for name in ("y", "mean", "rstd", "a", "c")}

    def check(self, r):
        norm.check_forward(self.dtype, self.x, self.weight, self.bias, r["y"], r["mean"], r["rstd"])
        w4.check(r["a"], r["y"], self.up, self.up_scales, self.up_zeros, self.group)
        w4.check(r["c"], r["a"], self.down, self.down_scales, None, self.group)


def run(program):
    program.enqueue()
    program.ctx.synchronize()
    return program.results()


@pytest.mark.parametrize("rows, vocab, width, dtype", [(130, 1500, 256, "bfloat16"), (700, 611, 333, "float16"),
                                                       (1, 1000, 64, "bfloat16")])
def test_training_step(rows, vocab, width, dtype, gpu_ctx) -> None:
    step = TrainingStep(gpu_ctx, rows, vocab, width, dtype)
    first = run(step)
    step.check(first)
    for name, again in run(step).items():
        assert np.array_equal(again, first[name]), name


@pytest.mark.parametrize("m, width, inner, group, dtype", [(1, 512, 2048, 128, "bfloat16"), (7, 1031, 700, 32, "float16"),
                                                           (40, 768, 3000, 64, "bfloat16")])
def test_tokens(m, width, inner, group, dtype, gpu_ctx) -> None:
    token = Token(gpu_ctx, m, width, inner, group, dtype)
    first = run(token)
    token.check(first)
    for name, again in run(token).items():
        assert np.array_equal(again, first[name]), name


def test_calls_of_different_sizes_share_a_context(gpu_ctx) -> None:
    """The scratch grows and is used by one operator after another, with nothing waiting in between."""
    programs = [Token(gpu_ctx, 1, 256, 512, 64, "bfloat16"), TrainingStep(gpu_ctx, 64, 700, 128, "bfloat16"),
                Token(gpu_ctx, 33, 512, 6000, 128, "float16"), TrainingStep(gpu_ctx, 300, 2000, 200, "float16")]
    for p in programs * 2:
        p.enqueue()
    gpu_ctx.synchronize()
    for p in programs:
        p.check(p.results())


def test_two_contexts_at_once() -> None:
    """Each context has its stream and its scratch; two threads enqueue on one each."""
    contexts = [cuda.Context(0), cuda.Context(0)]
    programs = [[Token(c, 5, 512, 3000, 64, "bfloat16"), TrainingStep(c, 200, 1500, 256, "bfloat16")] for c in contexts]
    alone = [[run(p) for p in mine] for mine in programs]

    def work(mine):
        for _ in range(5):
            for p in mine:
                p.enqueue()
        mine[0].ctx.synchronize()

    threads = [threading.Thread(target=work, args=(mine,)) for mine in programs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for mine, before in zip(programs, alone):
        for p, r in zip(mine, before):
            after = p.results()
            assert all(np.array_equal(after[name], r[name]) for name in r)
            p.check(after)


def test_a_call_that_finds_no_memory_leaves_the_next_one_alone(gpu_ctx) -> None:
    """2^24 rows by 2^20 columns leave a partial pair per row and 128 columns: more than any GPU holds. The call is
    refused before anything is launched, and its error is not read as the next launch's."""
    h, w = cuda.DeviceBuffer(gpu_ctx, (1 << 24, 1), np.float16), cuda.DeviceBuffer(gpu_ctx, (1 << 20, 1), np.float16)
    t = cuda.DeviceBuffer(gpu_ctx, (1 << 24,), np.int32)
    f, g = (cuda.DeviceBuffer(gpu_ctx, (1 << 24,), np.float32) for _ in range(2))
    x, _, weight, bias = norm.inputs(7, 300, "float32", "float32", 51)
    bx, bw, bb = (norm.make(gpu_ctx, v) for v in (x, weight, bias))
    y, mean, rstd = norm.empty(gpu_ctx, x.shape, np.float32), norm.empty(gpu_ctx, (7,), np.float32), norm.empty(gpu_ctx, (7,), np.float32)
    with pytest.raises(DeviceError, match="OUT_OF_MEMORY"):
        gpu_ctx.linear_cross_entropy(h, w, t, f, g)
    gpu_ctx.layer_norm(bx, y, weight=bw, bias=bb, eps=norm.EPS, mean=mean, rstd=rstd)
    gpu_ctx.synchronize()
    norm.check_forward("float32", x, weight, bias, y.to_numpy(), mean.to_numpy(), rstd.to_numpy())
    step = TrainingStep(gpu_ctx, 33, 300, 64, "bfloat16")
    step.check(run(step))
