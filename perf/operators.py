"""The operators behind the last decoder layer, as cases to measure: the norm, the head in 8 bits, the loss over the head.

A case is a dict of plain values.  ``op`` says which operator it is:

* ``norm``  ``ops.rms_norm`` (``form`` ``rms``) or ``ops.layer_norm`` (``layer``, with a bias) over ``cols`` columns of ``rows``
            tokens; ``train`` adds the gradients of the input, the weight and the bias.
* ``int8``  ``ops.int8_linear_forward``: 16-bit activations, quantised with a scale for each token within the call, times 8-bit
            weights with a scale for each output channel.
* ``loss``  ``ops.linear_cross_entropy``: the cross entropy of ``tokens`` targets over a vocabulary of ``vocab`` words, from
            ``hidden`` columns and the weight of the head; ``ignored`` of the tokens have no target.  ``train`` adds the gradients
            of both, ``reduction`` is the loss's.

``own`` chooses between the operators written out in elementary operations (false) and the calls above (true).
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
IGNORE = -100


def listed():
    return [
        # the norm in front of the head for one decoded token: call overhead and launch latency
        dict(name="rms-1x4096", op="norm", form="rms", rows=1, cols=4096, dtype="bf16", train=False),
        # layer norm of a few sequences, a width that no vector load divides, with its gradients
        dict(name="layer-train-517x1003", op="norm", form="layer", rows=517, cols=1003, dtype="fp16", train=True),
        # a training batch of 4096 tokens at the width of an 8B model
        dict(name="rms-train-4096x4096", op="norm", form="rms", rows=4096, cols=4096, dtype="bf16", train=True),
        # a large batch: bandwidth
        dict(name="layer-train-16384x5120", op="norm", form="layer", rows=16384, cols=5120, dtype="bf16", train=True),
        # sizes that nothing divides, with a bias
        dict(name="int8-1003x777-t37", op="int8", N=1003, V=777, tokens=37, dtype="fp16", bias=True),
        # the head of a decode step (Qwen3-8B vocabulary)
        dict(name="int8-151936x4096-t1", op="int8", N=4096, V=151936, tokens=1, dtype="bf16", bias=False),
        # sixteen sequences on a small model's head (Llama-3.2-1B)
        dict(name="int8-128256x2048-t16", op="int8", N=2048, V=128256, tokens=16, dtype="bf16", bias=False),
        # a prompt through a projection of an 8B model: tensor-core bound
        dict(name="int8-12288x4096-t2048", op="int8", N=4096, V=12288, tokens=2048, dtype="bf16", bias=False),
        # a handful of tokens on a toy vocabulary
        dict(name="loss-train-1003x512-t77", op="loss", hidden=512, vocab=1003, tokens=77, ignored=0.3, dtype="fp16",
             reduction="mean", train=True),
        # perplexity: the loss of every token of a window on a small model's head
        dict(name="loss-128256x2048-t512", op="loss", hidden=2048, vocab=128256, tokens=512, ignored=0.0, dtype="bf16",
             reduction="none", train=False),
        # a training step of the head with a small vocabulary (Llama-2-7B), prompts without a target
        dict(name="loss-train-32000x4096-t4096", op="loss", hidden=4096, vocab=32000, tokens=4096, ignored=0.25, dtype="fp16",
             reduction="mean", train=True),
        # and with a large one (Qwen3-8B)
        dict(name="loss-train-151936x4096-t2048", op="loss", hidden=4096, vocab=151936, tokens=2048, ignored=0.1, dtype="bf16",
             reduction="sum", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _up(v, m):
    return max(m, (v + m - 1) // m * m)


def draw(rng):
    most = {op: max((work(c) for c in listed() if c["op"] == op), key=lambda w: (w["flops"], w["bytes"])) for op in ("norm", "int8", "loss")}
    while True:
        c = _draw(rng)
        w, m = work(c), most[c["op"]]
        if w["flops"] <= m["flops"] and w["bytes"] <= (m["bytes"] if c["op"] == "norm" else 2.6e9):
            return c


def _draw(rng):
    dtype, op = rng.choice(["fp16", "bf16"]), rng.choice(["norm", "int8", "loss"])
    if op == "norm":
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.7:
            cols = _up(cols, 64)
        return dict(op=op, form=rng.choice(["rms", "layer"]), rows=_log(rng, 1, 32768), cols=cols, dtype=dtype, train=rng.random() < 0.6)
    if op == "int8":
        N, V = _log(rng, 256, 14336), _log(rng, 256, 152000)
        if rng.random() < 0.7:
            N, V = _up(N, 64), _up(V, 64)
        return dict(op=op, N=N, V=V, tokens=_log(rng, 1, 4096), dtype=dtype, bias=rng.random() < 0.3)
    return dict(op=op, hidden=_up(_log(rng, 256, 8192), 8), vocab=_log(rng, 256, 152000), tokens=_log(rng, 1, 4096),
                ignored=rng.choice([0.0, round(rng.uniform(0.0, 0.9), 2)]), dtype=dtype, reduction=rng.choice(["mean", "sum", "none"]),
                train=rng.random() < 0.6)


@torch.no_grad()
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda")
    rand = lambda *shape: torch.rand(shape, generator=gen, device="cuda")
    dtype, op = DTYPES[case["dtype"]], case["op"]
    state = dict(case, op=op)
    if op == "norm":
        rows, cols, layer = case["rows"], case["cols"], case["form"] == "layer"
        # a residual stream: tokens of different magnitude, an offset, a few columns that stand out
        x = randn(rows, cols) * (0.5 + 3 * rand(rows, 1)) + 0.1
        x[:, torch.randint(cols, (4,), generator=gen, device="cuda")] *= 10
        state.update(x=x.to(dtype), w=(1 + 0.2 * randn(cols)).to(dtype), b=(0.1 * randn(cols)).to(dtype) if layer else None,
                     dy=randn(rows, cols).to(dtype) if case["train"] else None, eps=1e-5 if layer else 1e-6)
        if case["train"]:
            state["leaves"] = [state[k].requires_grad_() for k in ("x", "w", "b") if state[k] is not None]
    elif op == "int8":
        N, V, T = case["N"], case["V"], case["tokens"]
        # weights as ops.quantize_int8 lays them out: rows at multiples of 16 bytes
        w = torch.zeros((V, _up(N, 16)), dtype=torch.int8, device="cuda")
        for v in range(0, V, 16384):
            w[v:v + 16384, :N] = randn(min(16384, V - v), N).mul_(32).round_().clamp_(-127, 127).to(torch.int8)
        state.update(x=randn(T, N).to(dtype), w=w[:, :N], ws=(0.02 / 32) * (0.5 + rand(V)),
                     b=randn(V).mul_(0.1).to(dtype) if case["bias"] else None)
    else:
        N, V, T = case["hidden"], case["vocab"], case["tokens"]
        w = torch.empty((V, N), dtype=dtype, device="cuda")
        for v in range(0, V, 16384):
            w[v:v + 16384] = randn(min(16384, V - v), N).mul_(1.28 / math.sqrt(N)).to(dtype)
        targets = torch.randint(V, (T,), generator=gen, device="cuda")
        # hidden states that know something of their targets: probabilities from a guess to near certainty
        h = randn(T, N) + w[targets].float() * (8 * rand(T, 1))
        targets[rand(T) < case["ignored"]] = IGNORE
        targets[0] = V - 1
        state.update(h=h.to(dtype), w=w, targets=targets)
        if case["train"]:
            g = rand(T) + 0.5 if case["reduction"] == "none" else torch.ones((), device="cuda")
            if case["dtype"] == "fp16":
                g *= 1024           # loss scaling, without which fp16 gradients are subnormal
            state.update(h=state["h"].requires_grad_(), w=w.requires_grad_(), g=g)
    return state


def run(state):
    op = state["op"]
    if own:
        from nanoquant_b200 import ops
        if op == "norm":
            if state["form"] == "rms":
                y = ops.rms_norm(state["x"], state["w"], eps=state["eps"])
            else:
                y = ops.layer_norm(state["x"], state["w"], state["b"], eps=state["eps"])
            return [y.detach(), *torch.autograd.grad(y, state["leaves"], state["dy"])] if state["train"] else y
        if op == "int8":
            return ops.int8_linear_forward(state["x"], state["w"], state["ws"], state["b"])
        loss = ops.linear_cross_entropy(state["h"], state["w"], state["targets"], ignore_index=IGNORE, reduction=state["reduction"])
        return [loss.detach(), *torch.autograd.grad(loss, (state["h"], state["w"]), state["g"])] if state["train"] else loss
    with torch.no_grad():
        return {"norm": _plain_norm, "int8": _plain_int8, "loss": _plain_loss}[op](state)


def _plain_norm(s):
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    layer = s["form"] == "layer"
    c = x - x.mean(1, keepdim=True) if layer else x
    rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + s["eps"])
    xhat = c * rstd
    y = xhat * w
    if layer:
        y = y + s["b"].float()
    if not s["train"]:
        return y.to(dtype)
    dy = s["dy"].float()
    g = dy * w
    dx = g - xhat * (g * xhat).mean(1, keepdim=True)
    if layer:
        dx = dx - g.mean(1, keepdim=True)
    out = [y.to(dtype), (dx * rstd).to(dtype), (dy * xhat).sum(0).to(dtype)]
    return out + [dy.sum(0).to(dtype)] if layer else out


def _plain_int8(s):
    x = s["x"].double()                         # (32 bits would decide between two whole numbers where x / scale lies halfway)
    scale = x.abs().amax(1, keepdim=True) / 127
    q = torch.where(scale > 0, torch.round(x / scale), torch.zeros_like(x))
    y = q @ s["w"].double().T                   # whole numbers beyond 2^24
    y = y * scale * s["ws"].double()
    if s["b"] is not None:
        y = y + s["b"].double()
    return y.to(s["x"].dtype)


def _plain_loss(s):
    h, w, t, dtype = s["h"].float(), s["w"].float(), s["targets"], s["h"].dtype
    live = t != IGNORE
    col = torch.where(live, t, torch.zeros_like(t))[:, None]
    logits = h @ w.T
    top = logits.amax(1, keepdim=True)
    p = torch.exp(logits - top)
    total = p.sum(1, keepdim=True)
    loss = torch.where(live, (torch.log(total) + top - logits.gather(1, col))[:, 0], torch.zeros_like(top[:, 0]))
    del logits
    count = live.sum()
    out = loss if s["reduction"] == "none" else loss.sum() if s["reduction"] == "sum" else (loss.double().sum() / count).float()
    if not s["train"]:
        return out
    g = s["g"].expand(len(t)) if s["reduction"] != "mean" else (s["g"] / count).expand(len(t))
    g = torch.where(live, g, torch.zeros_like(g))[:, None]
    p *= g / total
    p.scatter_add_(1, col, -g)
    return [out, (p @ w).to(dtype), (p.T @ h).to(dtype)]


def work(case):
    """Every input once, every output once, and the products: one for the logits, one for each gradient."""
    op = case["op"]
    if op == "norm":
        rows, cols, layer = case["rows"], case["cols"], case["form"] == "layer"
        vectors = 2 * cols * (2 if layer else 1)
        if case["train"]:       # x, dy in; y, dx out; the weight (and bias) in, their gradients out
            return dict(bytes=8 * rows * cols + 2 * vectors, flops=(16 if layer else 12) * rows * cols)
        return dict(bytes=4 * rows * cols + vectors, flops=(6 if layer else 4) * rows * cols)
    if op == "int8":
        N, V, T = case["N"], case["V"], case["tokens"]
        return dict(bytes=V * N + 4 * V + 2 * T * (N + V) + (2 * V if case["bias"] else 0), flops=2 * T * N * V)
    N, V, T = case["hidden"], case["vocab"], case["tokens"]
    outer = 4 * T if case["reduction"] == "none" else 4
    if case["train"]:
        return dict(bytes=4 * (T + V) * N + 8 * T + 2 * outer, flops=6 * T * N * V)
    return dict(bytes=2 * (T + V) * N + 8 * T + outer, flops=2 * T * N * V)


@torch.no_grad()
def exact(case, seed):
    """The definitions, in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, w, n = s["x"].double(), s["w"].double(), case["cols"]
        layer = case["form"] == "layer"
        mean = x.sum(1) / n if layer else torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
        d = (x - mean[:, None])
        sigma = (d.square().sum(1) / n + s["eps"]).sqrt()[:, None]
        y = d / sigma * w + (s["b"].double() if layer else 0)
        if not case["train"]:
            return y
        dy = s["dy"].double()
        # y_j = w_j d_j / sigma; d sigma / d x_k = d_k / (n sigma)
        u = dy * w / sigma
        dx = u - d * ((u * d).sum(1, keepdim=True) / (n * sigma.square()))
        if layer:
            dx -= u.sum(1, keepdim=True) / n
        grads = [dx, (dy * (d / sigma)).sum(0)] + ([dy.sum(0)] if layer else [])
        return [y, *grads]
    if case["op"] == "int8":
        x = s["x"].double()
        unit = x.abs().max(1).values / 127
        unit[unit == 0] = 1
        q = (x / unit[:, None]).round()
        y = torch.empty((case["tokens"], case["V"]), dtype=torch.float64, device="cuda")
        for v in range(0, case["V"], 32768):
            y[:, v:v + 32768] = q @ s["w"][v:v + 32768].double().T
        y *= unit[:, None] * s["ws"].double()
        return y if s["b"] is None else y + s["b"].double()
    h, t, V, T = s["h"].double(), s["targets"], case["vocab"], case["tokens"]
    live = (t != IGNORE).nonzero()[:, 0]
    logits = torch.empty((T, V), dtype=torch.float64, device="cuda")
    for v in range(0, V, 32768):
        logits[:, v:v + 32768] = h @ s["w"][v:v + 32768].double().T
    lse = torch.logsumexp(logits, 1)
    loss = torch.zeros(T, dtype=torch.float64, device="cuda")
    loss[live] = lse[live] - logits[live, t[live]]
    out = {"none": loss, "sum": loss.sum(), "mean": loss.sum() / max(1, len(live))}[case["reduction"]]
    if not case["train"]:
        return out
    g = torch.zeros(T, dtype=torch.float64, device="cuda")
    g[live] = s["g"].double()[live] if case["reduction"] == "none" else s["g"].double() / (len(live) if case["reduction"] == "mean" else 1)
    d = logits.sub_(lse[:, None]).exp_().mul_(g[:, None])
    d[live, t[live]] -= g[live]
    dh, dw = torch.zeros_like(h), torch.empty((V, case["hidden"]), dtype=torch.float64, device="cuda")
    for v in range(0, V, 32768):
        dh += d[:, v:v + 32768] @ s["w"][v:v + 32768].double()
        dw[v:v + 32768] = d[:, v:v + 32768].T @ h
    return [out, dh, dw]
