"""The operators between the projections of a decoder layer, as cases to measure: head norms and rotation, the paged cache, attention.

A case is a dict of plain values; ``heads`` query heads share ``kv`` key and value heads of ``dim`` elements.  ``op`` says which operator it is:

* ``rope``    ``ops.qk_norm_rope``: queries and keys of ``tokens`` tokens, rotated by their positions (``rotary`` of the ``dim`` elements,
              neighbours or halves as pairs), behind an RMS norm of each head with ``norm``.
* ``append``  ``ops.append_kv``: keys (normed and rotated on the way) and values of up to ``new`` tokens for each of ``seqs`` sequences
              into a cache of pages of ``page`` tokens that holds up to ``cached`` of each; with ``queries`` the rotated queries come back.
* ``prompt``  ``ops.prompt_attention``: causal attention of up to ``new`` tokens for each of ``seqs`` packed sequences, over themselves, or
              (``page`` > 0) over a paged cache that holds up to ``cached`` earlier tokens of each as well; ``window`` > 0 limits how far back.
* ``decode``  ``ops.paged_attention``: one new token for each of ``seqs`` sequences over up to ``cached`` tokens in pages.

``own`` chooses between the operators written out in elementary operations (false) and the calls above (true).
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    qwen, llama = dict(heads=32, kv=8, dim=128), dict(heads=32, kv=8, dim=64)      # Qwen3-8B, Llama-3.2-1B
    return [
        # one decoded token of an 8B model with head norms: call overhead and launch latency
        dict(name="rope-1", op="rope", tokens=1, **qwen, rotary=128, norm=True, neighbours=False, dtype="bf16"),
        # a few prompts of a model that rotates half of each head, neighbours as pairs, odd head counts
        dict(name="rope-517-partial", op="rope", tokens=517, heads=15, kv=5, dim=96, rotary=48, norm=False, neighbours=True, dtype="fp16"),
        # a large batch of prompts: bandwidth
        dict(name="rope-8192", op="rope", tokens=8192, **qwen, rotary=128, norm=True, neighbours=False, dtype="bf16"),
        # a decode step of sixteen sequences: queries rotated, keys and values stored, one call
        dict(name="append-16x1", op="append", seqs=16, new=1, cached=1024, page=16, **qwen, norm=True, queries=True, dtype="bf16"),
        # prompts of a small model into an empty cache
        dict(name="append-6x4096", op="append", seqs=6, new=4096, cached=0, page=32, **llama, norm=False, queries=False, dtype="fp16"),
        # a handful of chat turns of odd lengths
        dict(name="prompt-9x197", op="prompt", seqs=9, new=197, cached=0, page=0, **llama, window=0, dtype="fp16"),
        # prompts of different lengths in one batch
        dict(name="prompt-8x2048", op="prompt", seqs=8, new=2048, cached=0, page=0, **qwen, window=0, dtype="bf16"),
        # one long document
        dict(name="prompt-1x16384", op="prompt", seqs=1, new=16384, cached=0, page=0, **qwen, window=0, dtype="bf16"),
        # the next piece of four prompts behind what the cache holds already
        dict(name="prompt-chunk-4x512", op="prompt", seqs=4, new=512, cached=4096, page=16, **qwen, window=0, dtype="bf16"),
        # a single user's chat: latency
        dict(name="decode-1x1000", op="decode", seqs=1, cached=1000, page=16, **qwen, window=0, dtype="bf16"),
        # a serving batch of different lengths, every query head with keys of its own (Llama-2-7B)
        dict(name="decode-32x4096", op="decode", seqs=32, cached=4096, page=64, heads=32, kv=32, dim=128, window=0, dtype="fp16"),
        # long contexts of a 70B model
        dict(name="decode-4x131072", op="decode", seqs=4, cached=131072, page=64, heads=64, kv=8, dim=128, window=0, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {op: [max(work(c)[k] for c in listed() if c["op"] == op) for k in ("bytes", "flops")] for op in ("rope", "append", "prompt", "decode")}
    while True:
        c = _draw(rng)
        w, (b, f) = work(c), most[c["op"]]
        # (the plain form of a prompt keeps all scores of padded sequences)
        scores = c["seqs"] * c["heads"] * c["new"] * (c["new"] + c["cached"]) if c["op"] == "prompt" else 0
        if w["bytes"] <= b and w["flops"] <= f and scores <= 32 * 16384 ** 2:
            return c


def _draw(rng):
    op = rng.choice(["rope", "append", "prompt", "prompt", "decode", "decode"])
    kv = rng.choice([1, 2, 4, 5, 8, 8, 16, 32])
    dim = rng.choice([64, 64, 128, 128, 128, 80, 96, 192, 256])
    c = dict(op=op, heads=kv * rng.choice([1, 2, 3, 4, 4, 7, 8]), kv=kv, dim=dim, dtype=rng.choice(["fp16", "bf16"]))
    page = rng.choice([16, 32, 64, 128])
    window = _log(rng, 16, 4096) if rng.random() < 0.2 else 0
    if op == "rope":
        return dict(c, tokens=_log(rng, 1, 16384), rotary=rng.choice([dim, dim, dim // 2]), norm=rng.random() < 0.5, neighbours=rng.random() < 0.3)
    if op == "append":
        step = rng.random() < 0.5
        return dict(c, seqs=_log(rng, 1, 256 if step else 16), new=1 if step else _log(rng, 2, 8192), cached=_log(rng, 1, 1024), page=page,
                    norm=rng.random() < 0.5, queries=step)
    if op == "prompt":
        behind = rng.random() < 0.4
        return dict(c, seqs=_log(rng, 1, 24), new=_log(rng, 1, 16384), cached=_log(rng, 1, 16384) if behind else 0, page=page if behind else 0, window=window)
    return dict(c, seqs=_log(rng, 1, 256), cached=_log(rng, 1, 131072), page=page, window=window)


def _lengths(case):
    """(new tokens, tokens in the cache before) of each sequence: the longest, and others down to a sixteenth of it."""
    rng = random.Random("%d %d %d" % (case["seqs"], case.get("new", 1), case["cached"]))
    some = lambda n: [n] + [_log(rng, max(1, n // 16), n) for _ in range(case["seqs"] - 1)] if n else [0] * case["seqs"]
    new = some(case.get("new", 0))
    return new, some(case["cached"])


@torch.no_grad()
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda")
    rand = lambda *shape: torch.rand(shape, generator=gen, device="cuda")
    dtype, op, H, K, D = DTYPES[case["dtype"]], case["op"], case["heads"], case["kv"], case["dim"]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    state = dict(case)
    new, before = ([case["tokens"]], [0]) if op == "rope" else _lengths(case)
    T = len(before) if op == "decode" else sum(new)
    # what the projections give, side by side in one buffer; heads of different sharpness, as the logits of real ones are
    qkv = randn(T, H + 2 * K, D)
    qkv[:, :H] *= 0.5 + 2 * rand(H, 1)
    qkv = qkv.to(dtype).view(T, (H + 2 * K) * D)
    q, k, v = qkv[:, :H * D].view(T, H, D), qkv[:, H * D:(H + K) * D].view(T, K, D), qkv[:, (H + K) * D:].view(T, K, D)
    state.update(q=q, k=k, v=v)
    if op == "rope":
        far = torch.randint(131072, (1,), generator=gen, device="cuda")          # a place in a long context
        state["positions"] = (far + torch.arange(T, device="cuda")).int()
    if op in ("rope", "append"):
        R = case.get("rotary", D)
        state["inv_freq"] = 1e6 ** (torch.arange(0, R, 2, device="cuda").float() / -R)
        state["wq"], state["wk"] = ((1 + 0.2 * randn(D)).to(dtype) if case["norm"] else None for _ in range(2))
    if op == "prompt":
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        state.update(cu=ints(starts), starts=starts, new_lengths=new)
    if op != "rope" and case["page"]:
        page = case["page"]
        pages = [(a + b + page - 1) // page for a, b in zip(new, before)]
        total = sum(pages) + 3
        cache = [torch.empty((total, page, K, D), dtype=dtype, device="cuda") for _ in range(2)]
        for c in cache:
            for i in range(0, total, 8192):
                c[i:i + 8192] = randn(*c[i:i + 8192].shape).to(dtype)
        order, table, at = torch.randperm(total, generator=gen, device="cuda").int(), torch.zeros((len(new), max(pages)), dtype=torch.int32, device="cuda"), 0
        for i, n in enumerate(pages):
            table[i, :n] = order[at:at + n]
            at += n
        lengths = [a + b for a, b in zip(new, before)]
        state.update(k_cache=cache[0], v_cache=cache[1], table=table, lengths=ints(lengths), longest=max(lengths))
        if op == "append":
            state["sequences"] = torch.repeat_interleave(ints(list(range(len(new)))), ints(new))
            state["positions"] = torch.cat([torch.arange(b, b + a, device="cuda") for a, b in zip(new, before)]).int()
    return state


def run(state):
    op = state["op"]
    if own:
        from nanoquant_b200 import ops
        s = state
        with torch.no_grad():
            if op == "rope":
                return ops.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], s["wq"], s["wk"], eps=EPS, interleaved=s["neighbours"])
            if op == "append":
                q = ops.append_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["positions"], s["sequences"], s["inv_freq"], s["wk"],
                                  q=s["q"] if s["queries"] else None, q_weight=s["wq"] if s["queries"] else None, eps=EPS)
                return [s["k_cache"], s["v_cache"]] + ([q] if s["queries"] else [])
            if op == "prompt":
                if s["page"]:
                    return ops.prompt_attention(s["q"], s["k_cache"], s["v_cache"], s["cu"], block_table=s["table"], lengths=s["lengths"], window=s["window"] or None)
                return ops.prompt_attention(s["q"], s["k"], s["v"], s["cu"], window=s["window"] or None)
            return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], window=s["window"] or None)
    with torch.no_grad():
        return {"rope": _plain_rope, "append": _plain_append, "prompt": _plain_prompt, "decode": _plain_decode}[op](state)


def _plain_turned(x, w, angles, neighbours):
    """Heads, normed with ``w`` if there is one, then rotated: [T, heads, D] in 32 bits from any type; angles [T, pairs] in 64."""
    x = x.float()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(2, keepdim=True) + EPS) * w.float()
    pairs = angles.shape[1]
    cos, sin = torch.cos(angles).float()[:, None], torch.sin(angles).float()[:, None]
    a, b = (x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) if neighbours else (x[..., :pairs], x[..., pairs:2 * pairs])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, v), 3).flatten(2) if neighbours else torch.cat((u, v), 2)
    return torch.cat((turned, x[..., 2 * pairs:]), 2)


def _plain_rope(s):
    angles = s["positions"].double()[:, None] * s["inv_freq"].double()
    return tuple(_plain_turned(s[x], s["w" + x], angles, s["neighbours"]).to(s[x].dtype) for x in ("q", "k"))


def _plain_append(s):
    dtype, pos = s["k"].dtype, s["positions"].long()
    angles = s["positions"].double()[:, None] * s["inv_freq"].double()
    page, slot = s["table"][s["sequences"].long(), pos // s["page"]].long(), pos % s["page"]
    s["k_cache"][page, slot] = _plain_turned(s["k"], s["wk"], angles, False).to(dtype)
    s["v_cache"][page, slot] = s["v"]
    return [s["k_cache"], s["v_cache"]] + ([_plain_turned(s["q"], s["wq"], angles, False).to(dtype)] if s["queries"] else [])


def _plain_attention(q, k, v, seen):
    """q [B, Lq, H, D], k and v [B, Lk, K, D], seen [B, Lq, Lk]: [B, Lq, H, D] in 32 bits."""
    B, n, H, D = q.shape
    K = k.shape[2]
    q = q.float().view(B, n, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(B, K, H // K * n, D) * D ** -0.5
    p = torch.matmul(q, k.float().permute(0, 2, 3, 1)).view(B, K, H // K, n, -1)
    p.masked_fill_(~seen[:, None, None], -math.inf)
    p.sub_(p.amax(4, keepdim=True).clamp_(min=-1e30)).exp_()
    total = p.sum(4, keepdim=True)
    o = torch.matmul(p.view(B, K, H // K * n, -1), v.float().permute(0, 2, 1, 3)).view(B, K, H // K, n, D) / total.clamp_(min=1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D)


def _plain_prompt(s):
    dtype, n, cu = s["q"].dtype, s["new"], s["cu"].long()
    step = torch.arange(n, device="cuda")
    count = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + step).clamp(max=len(s["q"]) - 1)                  # tokens of padded sequences
    if s["page"]:
        k, v = (s[c][s["table"].long()].flatten(1, 2)[:, :s["longest"]] for c in ("k_cache", "v_cache"))
        length = s["lengths"].long()
    else:
        k, v, length = s["k"][at], s["v"][at], count
    row, col = (length - count)[:, None, None] + step[:, None], torch.arange(k.shape[1], device="cuda")
    seen = (col <= row) & (col < length[:, None, None])
    if s["window"]:
        seen &= col > row - s["window"]
    o = _plain_attention(s["q"][at], k, v, seen)
    token = torch.arange(len(s["q"]), device="cuda")
    of = (token[:, None] >= cu[1:]).sum(1)
    return o[of, token - cu[of]].to(dtype)


def _plain_decode(s):
    k, v = (s[c][s["table"].long()].flatten(1, 2)[:, :s["longest"]] for c in ("k_cache", "v_cache"))
    length, col = s["lengths"].long()[:, None, None], torch.arange(k.shape[1], device="cuda")
    seen = col < length
    if s["window"]:
        seen &= col >= length - s["window"]
    return _plain_attention(s["q"][:, None], k, v, seen)[:, 0].to(s["q"].dtype)


def work(case):
    """Every input once, every output once, and the two products of the pairs of tokens that see each other."""
    op, H, K, D = case["op"], case["heads"], case["kv"], case["dim"]
    if op == "rope":
        T = case["tokens"]
        return dict(bytes=4 * T * (H + K) * D + 4 * T + 2 * case["rotary"], flops=(7 if case["norm"] else 3) * T * (H + K) * D)
    new, before = _lengths(case)
    if op == "append":
        T, moved = sum(new), 2 * K + (H if case["queries"] else 0)
        return dict(bytes=4 * T * moved * D + 12 * T, flops=(7 if case["norm"] else 3) * T * (moved - K) * D)
    window = case["window"] or 1 << 40
    if op == "decode":
        seen = sum(min(b, window) for b in before)
        return dict(bytes=4 * seen * K * D + 4 * case["seqs"] * H * D + 4 * seen // case["page"], flops=4 * seen * H * D)
    # row i of a sequence sees min(b + i + 1, window) tokens
    pairs = 0
    for a, b in zip(new, before):
        full = min(max(0, window - b), a)                       # rows that see everything before them
        pairs += full * b + full * (full + 1) // 2 + (a - full) * min(window, 1 << 39)
    tokens = sum(min(a + b, a + window) for a, b in zip(new, before))
    return dict(bytes=4 * sum(new) * H * D + 4 * tokens * K * D, flops=4 * pairs * H * D)


@torch.no_grad()
def exact(case, seed):
    """The definitions, in 64 bits."""
    s = prepare(case, seed)
    op, H, K, D = case["op"], case["heads"], case["kv"], case["dim"]

    def turned(x, w, neighbours=False):
        x = x.double()
        if w is not None:
            x = w.double() * x * (x.square().sum(-1, keepdim=True) / D + EPS).rsqrt()
        # pairs as complex numbers, times exp(i position frequency)
        angle = torch.outer(s["positions"].double(), s["inv_freq"].double())
        n = angle.size(1)
        first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if neighbours else (slice(0, n), slice(n, 2 * n))
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * torch.polar(torch.ones_like(angle), angle).unsqueeze(1)
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    if op == "rope":
        return turned(s["q"], s["wq"], case["neighbours"]), turned(s["k"], s["wk"], case["neighbours"])
    if op == "append":
        k64, v64, key = s["k_cache"].double(), s["v_cache"].double(), turned(s["k"], s["wk"])
        flat = [c.view(-1, K, D) for c in (k64, v64)]
        where = s["table"].long()[s["sequences"].long()].gather(1, (s["positions"].long() // case["page"])[:, None])[:, 0] * case["page"] + s["positions"].long() % case["page"]
        flat[0].index_copy_(0, where, key)
        flat[1].index_copy_(0, where, s["v"].double())
        return [k64, v64] + ([turned(s["q"], s["wq"])] if case["queries"] else [])
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    new, before = _lengths(case)
    window = case["window"] or 1 << 40
    at = 0
    for i in range(case["seqs"]):
        rows = 1 if op == "decode" else new[i]
        length = before[i] if op == "decode" else new[i] + before[i]
        if case["page"]:
            pages = s["table"][i, :(length + case["page"] - 1) // case["page"]].long()
            keys, values = (s[c][pages].reshape(-1, K, D)[:length] for c in ("k_cache", "v_cache"))
        else:
            keys, values = s["k"][at:at + rows], s["v"][at:at + rows]
        for g in range(K):
            kg, vg = keys[:, g].double(), values[:, g].double()
            for r in range(0, rows, 2048):
                last = torch.arange(r, min(rows, r + 2048), device="cuda") + (length - rows)          # the token that a row is
                low, high = max(0, int(length - rows + r - window + 1)), int(last[-1]) + 1
                col = torch.arange(low, high, device="cuda")
                hidden = (col > last[:, None]) | (col <= last[:, None] - window)
                for h in range(g * (H // K), (g + 1) * (H // K)):
                    x = s["q"][at + r:at + r + len(last), h].double() @ kg[low:high].T / math.sqrt(D)
                    x.masked_fill_(hidden, -math.inf)
                    x -= x.logsumexp(1, keepdim=True)
                    out[at + r:at + r + len(last), h] = x.exp_() @ vg[low:high]
        at += rows
    return out
