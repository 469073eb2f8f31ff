"""Cases that measure the operators at the output end of a language model: layer norm with its
backward pass, softmax cross entropy of a linear layer over a large vocabulary with its gradients,
and products with weights held in 4 bits.

Every case runs in two ways. In the plain form `run` is elementary torch operations in 32 bits. With
`own` set it makes the calls a user of `hc.cuda` makes: `Context.layer_norm`,
`Context.layer_norm_backward`, `Context.linear_cross_entropy`, `Context.linear_cross_entropy_backward`
and `Context.gemm_w4` on `DeviceBuffer` objects (here: windows onto the torch tensors that hold the
inputs and the results).
"""

import math
import sys

import torch

own = False

EPS = 1e-5
IGNORE = -100
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # The norm before the output layer while one token is generated: latency.
        {"name": "norm_token", "op": "norm", "rows": 1, "cols": 4096, "type": "bfloat16", "offset": 0.0},
        # The same over a batch of ragged activations in float32, far from zero mean.
        {"name": "norm_ragged_f32", "op": "norm", "rows": 4095, "cols": 1031, "type": "float32", "offset": 3.0},
        # A training step's norm, forward and backward, at a usual width.
        {"name": "norm_step", "op": "norm_step", "rows": 16384, "cols": 4096, "type": "bfloat16", "offset": 0.0},
        # Wide rows, few of them.
        {"name": "norm_step_wide", "op": "norm_step", "rows": 1025, "cols": 16384, "type": "float16", "offset": 0.5},
        # Evaluation of a validation batch: the losses alone.
        {"name": "loss_eval", "op": "loss", "rows": 1024, "vocab": 32768, "width": 2048, "type": "bfloat16"},
        # A training step's loss with the gradients of the activations and of the vocabulary matrix.
        {"name": "loss_step", "op": "loss_step", "rows": 4096, "vocab": 32768, "width": 4096, "type": "bfloat16"},
        # The same with nothing round: rows, vocabulary and width all odd.
        {"name": "loss_step_ragged", "op": "loss_step", "rows": 1031, "vocab": 16411, "width": 1001, "type": "float16"},
        # A small model's step, or a short batch for fine-tuning.
        {"name": "loss_step_small", "op": "loss_step", "rows": 128, "vocab": 4099, "width": 512, "type": "bfloat16"},
        # One token through the output matrix held in 4 bits.
        {"name": "w4_token", "op": "w4", "m": 1, "n": 16384, "k": 8192, "group": 128, "zeros": False,
         "type": "bfloat16", "out": "bfloat16"},
        # Eight sequences at a time, with zero points, the logits kept in float32.
        {"name": "w4_batch", "op": "w4", "m": 8, "n": 16384, "k": 8192, "group": 64, "zeros": True,
         "type": "float16", "out": "float32"},
        # A small projection with an odd number of rows: latency.
        {"name": "w4_small", "op": "w4", "m": 1, "n": 1031, "k": 2048, "group": 32, "zeros": True,
         "type": "float16", "out": "float16"},
        # The widest batch of the skinny products.
        {"name": "w4_wide_batch", "op": "w4", "m": 64, "n": 8192, "k": 8192, "group": 128, "zeros": False,
         "type": "bfloat16", "out": "bfloat16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm_step", "loss", "loss_step", "w4", "w4"])
    if op in ("norm", "norm_step"):
        cols = _log(rng, 64, 16384)
        rows = _log(rng, 1, min(16384, (1 << 26) // cols))
        return {"op": op, "rows": rows, "cols": cols, "type": rng.choice(sorted(TYPES)),
                "offset": rng.choice([0.0, 0.5, 3.0])}
    if op in ("loss", "loss_step"):
        width = _log(rng, 64, 4096)
        vocab = _log(rng, 1000, 65000)
        rows = _log(rng, 16, min(4096, (1 << 39) // (width * vocab)))
        return {"op": op, "rows": rows, "vocab": vocab, "width": width, "type": rng.choice(["bfloat16", "float16"])}
    k = _log(rng, 128, 16384)
    n = _log(rng, 64, min(32768, (1 << 27) // k))
    kind = rng.choice(["bfloat16", "float16"])
    return {"op": op, "m": _log(rng, 1, 64), "n": n, "k": k, "group": rng.choice([32, 64, 128]),
            "zeros": rng.choice([True, False]), "type": kind, "out": rng.choice([kind, "float32"])}


def work(case):
    if case["op"] in ("norm", "norm_step"):
        size = 4 if case["type"] == "float32" else 2
        cells = case["rows"] * case["cols"]
        if case["op"] == "norm":
            return {"bytes": size * (2 * cells + 2 * case["cols"]) + 8 * case["rows"], "flops": 8 * cells}
        # x read and y written; then x and dy read and dx written
        return {"bytes": size * (5 * cells + 5 * case["cols"]) + 16 * case["rows"], "flops": 22 * cells}
    if case["op"] in ("loss", "loss_step"):
        product = 2 * case["rows"] * case["vocab"] * case["width"]
        inputs = 2 * (case["rows"] + case["vocab"]) * case["width"]
        if case["op"] == "loss":
            return {"bytes": inputs + 16 * case["rows"], "flops": product}
        return {"bytes": 2 * inputs + 28 * case["rows"], "flops": 3 * product}
    m, n, k = case["m"], case["n"], case["k"]
    groups = n * -(-k // case["group"])
    size = 4 if case["out"] == "float32" else 2
    return {"bytes": n * -(-k // 2) + groups * (3 if case["zeros"] else 2) + 2 * m * k + size * m * n,
            "flops": 2 * m * n * k}


# ---------------------------------------------------------------- what a program has in hand

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).add_(shift)

    s = {"case": case}
    if case["op"] in ("norm", "norm_step"):
        rows, cols = case["rows"], case["cols"]
        # Activations: a few channels much larger than the rest, rows of different size.
        channel = torch.exp(normal(cols, scale=0.5))
        s["x"] = (normal(rows, cols) * channel * torch.exp(normal(rows, 1, scale=0.3)) + case["offset"]).to(dtype)
        s["weight"] = normal(cols, scale=0.1, shift=1.0).to(dtype)
        s["bias"] = normal(cols, scale=0.1).to(dtype)
        s["y"] = torch.empty_like(s["x"])
        s["mean"], s["rstd"] = (torch.empty(rows, device="cuda") for _ in range(2))
        if case["op"] == "norm_step":
            s["dy"] = normal(rows, cols, scale=0.02).to(dtype)
            s["dx"] = torch.empty_like(s["x"])
            s["dweight"], s["dbias"] = torch.empty_like(s["weight"]), torch.empty_like(s["bias"])
    elif case["op"] in ("loss", "loss_step"):
        rows, vocab, width = case["rows"], case["vocab"], case["width"]
        s["w"] = normal(vocab, width, scale=1.0 / math.sqrt(width)).to(dtype)
        targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        # Some rows are nearly sure of their token, most are not.
        sure = torch.rand(rows, 1, generator=g, device="cuda") ** 4 * 12.0
        s["h"] = (normal(rows, width) + sure * s["w"][targets].float()).to(dtype)
        padding = torch.rand(rows, generator=g, device="cuda") < 1.0 / 16.0
        s["targets"] = torch.where(padding, torch.full_like(targets, IGNORE), targets)
        s["loss"], s["lse"] = (torch.empty(rows, device="cuda") for _ in range(2))
        if case["op"] == "loss_step":
            # The mean over the rows that count; float16 training scales its loss.
            scale = 1024.0 if case["type"] == "float16" else 1.0
            count = torch.clamp((~padding).sum(), min=1).float()
            s["dloss"] = torch.where(padding, torch.zeros((), device="cuda"), scale / count)
            s["dh"], s["dw"] = torch.empty_like(s["h"]), torch.empty_like(s["w"])
    else:
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // case["group"])
        s["a"] = normal(m, k).to(dtype)
        s["packed"] = torch.randint(0, 256, (n, -(-k // 2)), generator=g, device="cuda", dtype=torch.uint8)
        s["scales"] = (torch.rand(n, groups, generator=g, device="cuda") + 0.5).mul_(0.01).to(dtype)
        s["zeros"] = (torch.randint(6, 11, (n, groups), generator=g, device="cuda", dtype=torch.uint8)
                      if case["zeros"] else None)
        s["c"] = torch.empty(m, n, device="cuda", dtype=TYPES[case["out"]])
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    if op == "norm":
        return _plain_norm(state)[:3]
    if op == "norm_step":
        return _plain_norm_step(state)
    if op == "loss":
        return _plain_loss(state)[:2]
    if op == "loss_step":
        return _plain_loss_step(state)
    return _plain_w4(state)


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(dim=1, keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean(dim=1, keepdim=True) + EPS)
    normed = centred * rstd
    y = normed * s["weight"].float() + s["bias"].float()
    return y.to(s["x"].dtype), mean[:, 0], rstd[:, 0], normed


def _plain_norm_step(s):
    y, mean, rstd, normed = _plain_norm(s)
    dtype = s["x"].dtype
    dy = s["dy"].float()
    scaled = dy * s["weight"].float()
    dx = rstd[:, None] * (scaled - scaled.mean(dim=1, keepdim=True)
                          - normed * (scaled * normed).mean(dim=1, keepdim=True))
    return (y, mean, rstd, dx.to(dtype), (dy * normed).sum(dim=0).to(dtype), dy.sum(dim=0).to(dtype))


def _plain_loss(s):
    logits = s["h"].float() @ s["w"].float().t()
    largest = logits.max(dim=1).values
    lse = torch.log(torch.exp(logits - largest[:, None]).sum(dim=1)) + largest
    counts = s["targets"] != IGNORE
    at = torch.where(counts, s["targets"], torch.zeros_like(s["targets"]))
    loss = torch.where(counts, lse - logits.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
    return loss, lse, logits, counts, at


def _plain_loss_step(s):
    loss, lse, logits, counts, at = _plain_loss(s)
    grad = torch.exp(logits - lse[:, None])
    grad.scatter_add_(1, at[:, None], torch.full_like(lse, -1.0)[:, None])
    grad = grad * torch.where(counts, s["dloss"], torch.zeros_like(s["dloss"]))[:, None]
    dtype = s["h"].dtype
    return loss, lse, (grad @ s["w"].float()).to(dtype), (grad.t() @ s["h"].float()).to(dtype)


def _plain_w4(s):
    k, group = s["case"]["k"], s["case"]["group"]
    packed = s["packed"]
    q = torch.stack((packed & 15, packed >> 4), dim=2).reshape(packed.shape[0], -1)[:, :k].float()
    at = torch.arange(k, device=q.device) // group
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[:, at]
    weights = (q - zero) * s["scales"].float()[:, at]
    return (s["a"].float() @ weights.t()).to(s["c"].dtype)


def _own(s, op):
    ctx, b = s.get("own") or _wrap(s)
    if op in ("norm", "norm_step"):
        ctx.layer_norm(b["x"], b["y"], weight=b["weight"], bias=b["bias"], eps=EPS, mean=b["mean"], rstd=b["rstd"])
        if op == "norm":
            return s["y"], s["mean"], s["rstd"]
        ctx.layer_norm_backward(b["dy"], b["x"], b["dx"], mean=b["mean"], rstd=b["rstd"], weight=b["weight"],
                                dweight=b["dweight"], dbias=b["dbias"])
        return s["y"], s["mean"], s["rstd"], s["dx"], s["dweight"], s["dbias"]
    if op in ("loss", "loss_step"):
        ctx.linear_cross_entropy(b["h"], b["w"], b["targets"], b["loss"], b["lse"], ignore_index=IGNORE)
        if op == "loss":
            return s["loss"], s["lse"]
        ctx.linear_cross_entropy_backward(b["h"], b["w"], b["targets"], b["lse"], b["dloss"], dh=b["dh"], dw=b["dw"],
                                          ignore_index=IGNORE)
        return s["loss"], s["lse"], s["dh"], s["dw"]
    ctx.gemm_w4(b["a"], b["packed"], b["scales"], b["c"], group=s["case"]["group"], zeros=b.get("zeros"))
    return s["c"]


def _wrap(s):
    """The tensors as the framework's device buffers, made once for a state: they own nothing."""
    if "5_b200" not in sys.path:
        sys.path.insert(0, "5_b200")
    from hc import cuda

    ctx = cuda.default_context()
    buffers = {}
    for name, t in s.items():
        if isinstance(t, torch.Tensor):
            buffers[name] = cuda.DeviceBuffer.wrap(ctx, t.data_ptr(), tuple(t.shape), str(t.dtype).replace("torch.", ""))
    torch.cuda.synchronize()  # the library works on a stream of its own: the inputs are complete first
    s["own"] = (ctx, buffers)
    return s["own"]


# ---------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "norm_step"):
        x, weight, bias = s["x"].double(), s["weight"].double(), s["bias"].double()
        cols = case["cols"]
        mean = x.sum(1) / cols
        rstd = 1.0 / torch.sqrt(((x - mean[:, None]) ** 2).sum(1) / cols + EPS)
        normed = (x - mean[:, None]) * rstd[:, None]
        y = torch.addcmul(bias, normed, weight)
        if case["op"] == "norm":
            return y, mean, rstd
        dy = s["dy"].double()
        inner = torch.einsum("rc,c,rc->r", dy, weight, normed) / cols
        level = dy @ weight / cols
        dx = (dy * weight - level[:, None] - inner[:, None] * normed) * rstd[:, None]
        return y, mean, rstd, dx, torch.einsum("rc,rc->c", dy, normed), dy.sum(0)
    if case["op"] in ("loss", "loss_step"):
        h, w, targets = s["h"].double(), s["w"].double(), s["targets"]
        logits = torch.einsum("nd,vd->nv", h, w)
        lse = torch.logsumexp(logits, 1)
        keep = torch.nonzero(targets != IGNORE)[:, 0]
        loss = torch.zeros_like(lse)
        loss[keep] = lse[keep] - logits[keep, targets[keep]]
        if case["op"] == "loss":
            return loss, lse
        delta = torch.softmax(logits, 1)
        del logits
        delta[keep, targets[keep]] -= 1.0
        upstream = torch.zeros_like(lse)
        upstream[keep] = s["dloss"].double()[keep]
        delta *= upstream[:, None]
        return loss, lse, torch.einsum("nv,vd->nd", delta, w), torch.einsum("nv,nd->vd", delta, h)
    m, n, k, group = case["m"], case["n"], case["k"], case["group"]
    digits = torch.empty(n, 2 * s["packed"].shape[1], dtype=torch.float64, device="cuda")
    digits[:, 0::2] = torch.remainder(s["packed"], 16).double()
    digits[:, 1::2] = torch.div(s["packed"], 16, rounding_mode="floor").double()
    total = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    a, scales = s["a"].double(), s["scales"].double()
    for j in range(scales.shape[1]):
        span = slice(j * group, min(k, (j + 1) * group))
        zero = torch.full((n, 1), 8.0, dtype=torch.float64, device="cuda") if s["zeros"] is None else s["zeros"][:, j:j + 1].double()
        total += a[:, span] @ (digits[:, span] - zero).t() * scales[:, j]
    return total
