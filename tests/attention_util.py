"""Definitions in 64 bits of what stands between the projections of a decoder layer, and the errors that the arithmetic of the kernels allows."""
import math

import torch

DTYPES = [torch.float16, torch.bfloat16]
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}       # half a subnormal step


def rand(seed, *shape, dtype=None, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randn(shape, generator=g, device="cuda") * scale
    return t if dtype is None else t.to(dtype)


def turned(x, positions, inv_freq, weight=None, eps=1e-6, interleaved=False, scaling=1.0):
    """Heads [T, H, D], normed where there is a weight, rotated; and the sum of the magnitudes that each result is made of."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    if inv_freq is None:
        return x, x.abs()
    angle = positions.double()[:, None] * inv_freq.double()
    cos, sin, n = angle.cos()[:, None] * scaling, angle.sin()[:, None] * scaling, inv_freq.numel()
    i = torch.arange(n, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    y, mag = x.clone(), x.abs()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    mag[..., a] = (x[..., a] * cos).abs() + (x[..., b] * sin).abs()
    mag[..., b] = (x[..., b] * cos).abs() + (x[..., a] * sin).abs()
    return y, mag


def check_turned(got, want, mag, what="", far=0):
    """One rounding of the result; in fp32 before: the norm (sum of squares, division, root, two products: below 40 roundings for up to 256 elements, added pairwise in
    halves), the angle to 2^-24 of a turn (an error of 2 pi 2^-24 in cos and sin), two products and a sum.
    `far`: the largest angle, where fp64 itself rounds it: the kernel's product, 1 / (2 pi) and its product are each off by 2^-53 of it, the product here by one more."""
    u = torch.finfo(got.dtype).eps / 2
    bound = u * want.abs() + ((40 + 7 + 4) * 2.0 ** -24 + far * 2.0 ** -51) * mag + TINY[got.dtype]
    over = ((got.double() - want).abs() - bound * (1 + 2.0 ** -8)).max().item()
    assert over <= 0, (what, over)


def attention64(q, k, v, place, scale=None, window=None, causal=True):
    """q [n, H, D], k and v [L, K, D], place [n] of each query: (o, sum p |v|, sum |v| of what is seen)."""
    n, H, D = q.shape
    L, K = k.shape[:2]
    scale = D ** -0.5 if scale is None else scale
    col = torch.arange(L, device=q.device)
    seen = (col <= place[:, None]) if causal else torch.ones((n, L), dtype=torch.bool, device=q.device)
    if window:
        seen = seen & (col > place[:, None] - window)
    o, avg, all_v = (torch.zeros((n, H, D), dtype=torch.float64, device=q.device) for _ in range(3))
    for h in range(H):
        g = h // (H // K)
        s = q[:, h].double() @ k[:, g].double().T * scale
        s = s.masked_fill(~seen, -math.inf)
        p = torch.exp(s - s.amax(1, keepdim=True).clamp(min=-1e300)) if L else s
        total = p.sum(1, keepdim=True)
        p = torch.where(total > 0, p / total, torch.zeros_like(p)) if L else p
        x = v[:, g].double()
        x = torch.where(seen.any(0)[:, None], x, torch.zeros_like(x))          # what no query sees does not enter, whatever it is
        o[:, h], avg[:, h], all_v[:, h] = p @ x, p @ x.abs(), seen.double() @ x.abs()
    return o, avg, all_v


def check_attention(got, ref, what=""):
    """u: half a step of the 16-bit type.  Weights p rounded once, and their sum off by as much at most: 2 u of the average of |v|.  Scores and exponents
    in fp32: products of up to 256 columns on the tensor cores (16 at a time, cut off at 2^-23 of the largest: below 2^-18 of the sum of magnitudes, which the inputs
    here keep below 2^6 after scaling: 2^-12 of p at most, and of the sum: 2^-11 together; half of it for its sign).  The result rounded once.  fp16 weights
    below 2^-14 of the largest are off by 2^-25 of it."""
    o, avg, all_v = ref
    assert got.shape == o.shape, what
    if got.numel() == 0:
        return
    u = torch.finfo(got.dtype).eps / 2
    bound = u * o.abs() + (2 * u + 2.0 ** -12) * avg + TINY[got.dtype] * (1 + all_v)
    diff = (got.double() - o).abs()
    assert not torch.isnan(got).any(), what
    over = (diff - bound * (1 + 2.0 ** -8)).max().item()
    assert over <= 0, (what, over)


def paged(k, v, lengths, page, seed=0, order="pages", dtype=None, spare=3, width=None, fill=float("nan")):
    """Sequences' keys and values [L, K, D] in pages at random places: (k_cache, v_cache, table); what holds no token is `fill`."""
    g = torch.Generator().manual_seed(seed)
    K, D = k[0].shape[1:]
    need = [(n + page - 1) // page for n in lengths]
    total = sum(need) + spare
    shape = {"pages": (total, page, K, D), "heads": (total, K, page, D)}[order]
    caches = [torch.full(shape, fill, dtype=k[0].dtype, device="cuda") for _ in range(2)]
    views = [c if order == "pages" else c.transpose(1, 2) for c in caches]
    perm, at = torch.randperm(total, generator=g), 0
    table = torch.full((len(lengths), width or max(max(need), 1)), -7, dtype=torch.int32)       # (nobody may look at what holds nothing)
    for s, n in enumerate(lengths):
        mine = perm[at:at + need[s]]
        at += need[s]
        table[s, :need[s]] = mine.int()
        for c, x in zip(views, (k[s], v[s])):
            pad = torch.full((need[s] * page, K, D), fill, dtype=x.dtype, device="cuda")
            pad[:n] = x[:n]
            if need[s]:
                c[mine.cuda()] = pad.view(need[s], page, K, D)
    return views[0], views[1], table.cuda()
