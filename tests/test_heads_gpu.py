"""Head norms with the rotation (`ops.qk_norm_rope`) and the paged cache (`ops.append_kv`) against their definitions in 64 bits."""
import pytest
import torch

from tests.attention_util import DTYPES, check_turned, rand, turned

pytestmark = pytest.mark.gpu


def freqs(R, theta=1e6):
    return theta ** (torch.arange(0, R, 2, device="cuda").float() / -R)


def weights(D, dtype, kind, seed=9):
    if kind == "none":
        return None, None
    t = torch.float32 if kind == "fp32" else dtype
    return (1 + 0.2 * rand(seed, D)).to(t), (1 + 0.2 * rand(seed + 1, D)).to(t)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,K,D,R,interleaved,norm", [
    (1, 32, 8, 128, 128, False, "own"), (5, 32, 8, 64, 64, False, "none"), (37, 15, 5, 96, 48, True, "fp32"), (3, 1, 1, 8, 8, False, "own"), (2, 4, 2, 80, 20, False, "own"),
    (7, 6, 3, 80, 40, False, "fp32"), (9, 3, 1, 256, 256, False, "own"), (4, 71, 1, 64, 64, True, "own"), (2, 8, 8, 192, 96, False, "none"), (3, 8, 2, 80, 20, True, "own"),
    (130, 64, 8, 128, 64, False, "own"), (3, 4, 4, 128, 0, False, "own"), (2, 2, 1, 72, 66, False, "none"), (2, 5, 1, 24, 24, True, "fp32"), (3, 100, 30, 128, 128, True, "own")])
def test_against_definition(T, H, K, D, R, interleaved, norm, dtype):
    from nanoquant_b200 import ops

    qkv = rand(T, T, (H + 2 * K) * D, dtype=dtype)                       # views of one buffer, as a launch group gives them
    q, k = qkv[:, :H * D].view(T, H, D), qkv[:, H * D:(H + K) * D].view(T, K, D)
    wq, wk = weights(D, dtype, norm)
    f = freqs(R) if R else torch.empty(0, device="cuda")
    pos = torch.randint(0, 131072, (T,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    for positions in (pos, pos.int(), -pos):
        gq, gk = ops.qk_norm_rope(q, k, positions, f, wq, wk, eps=1e-5, interleaved=interleaved, scaling=1.25)
        assert gq.shape == q.shape and gq.is_contiguous() and gk.shape == k.shape and gk.dtype == dtype
        for got, x, w in ((gq, q, wq), (gk, k, wk)):
            check_turned(got, *turned(x, positions, f if R else None, w, 1e-5, interleaved, 1.25), (positions.dtype, w is not None))


@pytest.mark.parametrize("position", [0, 1, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 40 + 3])
def test_angles_of_far_positions(position):
    """The angle is formed and reduced in 64 bits: the error grows with the position by 2^-51 of it only."""
    from nanoquant_b200 import ops

    q = rand(0, 2, 4, 128, dtype=torch.bfloat16)
    pos, f = torch.tensor([position, -position], device="cuda"), freqs(128, 1e4)
    got = ops.qk_norm_rope(q, q[:, :1], pos, f)
    check_turned(got[0], *turned(q, pos, f), far=position)
    check_turned(got[1], *turned(q[:, :1], pos, f), far=position)


def test_layouts_and_leading_dimensions():
    """What is not read in place is copied: odd strides and addresses, expanded and reversed dimensions, weights at odd addresses."""
    from nanoquant_b200 import ops

    f, pos = freqs(64), torch.arange(12, device="cuda")
    base = rand(1, 12, 9, 67, dtype=torch.float16)
    w = rand(2, 65, dtype=torch.float16)[1:]
    for q in (base[:, :, 1:65], base[:, ::2, :64], base[:, :1, :64].expand(12, 4, 64), base.transpose(0, 1)[:, :, :64].contiguous().transpose(0, 1), rand(3, 64, 12, 4, dtype=torch.float16).permute(1, 2, 0)):
        k = q[:, :1]
        want = ops.qk_norm_rope(q.contiguous().clone(), k.contiguous().clone(), pos, f, w.clone(), w.clone())
        got = ops.qk_norm_rope(q, k, pos, f, w, w)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        got = ops.qk_norm_rope(q.unflatten(0, (3, 4)), k.unflatten(0, (3, 4)), pos.view(3, 4), f, w, w)
        assert all(torch.equal(a.flatten(0, 1), b) for a, b in zip(got, want)) and got[0].shape[:2] == (3, 4)
    neg = torch._neg_view(q)
    assert all(torch.equal(a, b) for a, b in zip(ops.qk_norm_rope(neg, neg[:, :1], pos, f, w, w), ops.qk_norm_rope(-q, -k, pos, f, w, w)))
    empty = ops.qk_norm_rope(q[:0], k[:0], pos[:0], f)
    assert empty[0].shape == (0, 4, 64)


def fill_cache(pages, page, K, D, dtype, order):
    shape = (pages, page, K, D) if order == "pages" else (pages, K, page, D)
    c = rand(5, *shape, dtype=dtype), rand(6, *shape, dtype=dtype)
    return c if order == "pages" else tuple(x.transpose(1, 2) for x in c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("order", ["pages", "heads"])
@pytest.mark.parametrize("H,K,D,page,norm,with_q", [(8, 2, 128, 16, "own", True), (6, 3, 64, 8, "none", False), (4, 4, 80, 32, "fp32", True), (2, 1, 256, 64, "own", False), (3, 1, 24, 16, "own", True)])
def test_append(H, K, D, page, norm, with_q, order, dtype):
    """Prompts of several sequences at once: what is stored, what comes back, and that nothing else is touched."""
    from nanoquant_b200 import ops

    starts, new = [0, 5, 100], [page + 3, 1, 2 * page]
    seqs = torch.tensor([s for s, n in enumerate(new) for _ in range(n)], dtype=torch.int32, device="cuda")
    pos = torch.tensor([b + i for b, n in zip(starts, new) for i in range(n)], dtype=torch.int32, device="cuda")
    T, width = len(pos), (100 + 2 * page + page - 1) // page
    table = torch.randperm(3 * width + 2, generator=torch.Generator().manual_seed(3))[:3 * width].view(3, width).int().cuda()
    cache = fill_cache(3 * width + 2, page, K, D, dtype, order)
    before = [c.clone() for c in cache]
    qkv = rand(7, T, (H + 2 * K) * D, dtype=dtype)
    q, k, v = (t.view(T, -1, D) for t in qkv.split([H * D, K * D, K * D], 1))
    wq, wk = weights(D, dtype, norm)
    f = freqs(D // 2 * 2)
    got = ops.append_kv(k, v, *cache, table, pos, seqs, f, wk, q=q if with_q else None, q_weight=wq if with_q else None)
    if with_q:
        check_turned(got, *turned(q, pos, f, wq))
    else:
        assert got is None
    at = table[seqs.long(), pos.long() // page].long(), pos.long() % page
    check_turned(cache[0][at], *turned(k, pos, f, wk))
    assert torch.equal(cache[1][at], v)
    for c, b in zip(cache, before):
        b[at] = c[at]
        assert torch.equal(c, b)


def test_append_without_rotation_and_one_token_each():
    from nanoquant_b200 import ops

    k, v = rand(1, 4, 2, 64, dtype=torch.float16), rand(2, 4, 2, 64, dtype=torch.float16)
    table = torch.tensor([[3, 0], [1, 2], [5, 4], [7, 6]], dtype=torch.int32, device="cuda")
    cache = fill_cache(8, 8, 2, 64, torch.float16, "pages")
    pos = torch.tensor([0, 15, 8, 7], device="cuda")
    version = cache[0]._version
    assert ops.append_kv(k, v, *cache, table, pos) is None
    at = table[torch.arange(4, device="cuda"), pos // 8].long(), pos % 8
    assert torch.equal(cache[0][at], k) and torch.equal(cache[1][at], v) and cache[0]._version > version


def test_places_that_are_not_there_store_nothing():
    """Padding, positions behind the table, sequences and pages that do not exist."""
    from nanoquant_b200 import ops

    T = 8
    k, v, q = (rand(s, T, 2, 64, dtype=torch.bfloat16) for s in range(3))
    table = torch.tensor([[1, -1], [99, 2], [2 ** 31 - 1, 8], [-2 ** 31, 0]], dtype=torch.int32, device="cuda")
    cache = fill_cache(8, 8, 2, 64, torch.bfloat16, "pages")
    before = [c.clone() for c in cache]
    pos = torch.tensor([-1, -2 ** 62, 8, 0, 16, 2 ** 62, 3, 0], device="cuda")
    seqs = torch.tensor([0, 1, 0, 1, 3, 3, -1, 4], dtype=torch.int32, device="cuda")
    f = freqs(64)
    got = ops.append_kv(k, v, *cache, table, pos, seqs, f, q=q)
    assert all(torch.equal(c, b) for c, b in zip(cache, before))
    assert (got[:2] == 0).all()
    check_turned(got[2:4], *turned(q[2:4], pos[2:4], f))
    pos[3] = 8                                                    # one that is there
    ops.append_kv(k, v, *cache, table, pos, seqs, f)
    assert torch.equal(cache[1][2, 0], v[3]) and not torch.equal(cache[0], before[0])


def test_special_values():
    """A head with a NaN or an infinity spoils itself alone; a head of zeros stays zero."""
    from nanoquant_b200 import ops

    q = rand(0, 3, 4, 64, dtype=torch.bfloat16)
    q[1, 2, 5], q[2, 0, 7], q[0, 1] = float("nan"), float("inf"), 0
    w, f, pos = torch.ones(64, device="cuda"), freqs(64), torch.arange(3, device="cuda")
    got = ops.qk_norm_rope(q, q[:, :1], pos, f, w, w)[0]
    bad = torch.isnan(got).any(-1)
    assert bad[1, 2] and bad[2, 0] and bad.sum() == 2 and (got[0, 1] == 0).all()


def test_refusals():
    from nanoquant_b200 import ops

    q, k, v = rand(0, 4, 8, 64, dtype=torch.float16), rand(1, 4, 2, 64, dtype=torch.float16), rand(2, 4, 2, 64, dtype=torch.float16)
    f, pos = freqs(64), torch.arange(4, device="cuda")
    w = torch.ones(64, device="cuda")
    cache = fill_cache(4, 8, 2, 64, torch.float16, "pages")
    table = torch.zeros((4, 1), dtype=torch.int32, device="cuda")
    for match, call in (
            ("CUDA", lambda: ops.qk_norm_rope(q.cpu(), k, pos, f)), ("Half or BFloat16", lambda: ops.qk_norm_rope(q.float(), k, pos, f)), ("k is", lambda: ops.qk_norm_rope(q, k.bfloat16(), pos, f)),
            ("k has shape", lambda: ops.qk_norm_rope(q, k[:3], pos, f)), ("multiple of 8", lambda: ops.qk_norm_rope(q[..., :60], k[..., :60], pos, f[:4])), ("positions", lambda: ops.qk_norm_rope(q, k, pos[:3], f)),
            ("positions", lambda: ops.qk_norm_rope(q, k, pos.float(), f)), ("inv_freq", lambda: ops.qk_norm_rope(q, k, pos, f.half())), ("inv_freq", lambda: ops.qk_norm_rope(q, k, pos, freqs(66))),
            ("inv_freq", lambda: ops.qk_norm_rope(q, k, pos, None)), ("q_weight", lambda: ops.qk_norm_rope(q, k, pos, f, w[:32])), ("one type", lambda: ops.qk_norm_rope(q, k, pos, f, w, w.half())),
            ("positions", lambda: ops.qk_norm_rope(q, k, pos.cpu(), f)), ("multiple of 8", lambda: ops.qk_norm_rope(rand(0, 4, 1, 264, dtype=torch.float16), rand(0, 4, 1, 264, dtype=torch.float16), pos, f)),
            ("v has shape", lambda: ops.append_kv(k, v[:, :1], *cache, table, pos)), ("k_cache", lambda: ops.append_kv(k, v, cache[0][:, :6], cache[1][:, :6], table, pos)),
            ("k_cache", lambda: ops.append_kv(k, v, cache[0].bfloat16(), cache[1], table, pos)), ("k_cache has shape", lambda: ops.append_kv(k, v, cache[0][:, :, :1], cache[1][:, :, :1], table, pos)),
            ("v_cache", lambda: ops.append_kv(k, v, cache[0], cache[1][:3], table, pos)), ("block_table", lambda: ops.append_kv(k, v, *cache, table.long(), pos)),
            ("block_table", lambda: ops.append_kv(k, v, *cache, table[:0], pos)), ("sequences", lambda: ops.append_kv(k, v, *cache, table, pos, pos)), ("q_weight needs", lambda: ops.append_kv(k, v, *cache, table, pos, q_weight=w)),
            ("in place", lambda: ops.append_kv(k, v, rand(0, 4, 8, 2, 65, dtype=torch.float16)[..., :64], cache[1], table, pos)), ("q has shape", lambda: ops.append_kv(k, v, *cache, table, pos, q=q[:3]))):
        with pytest.raises(RuntimeError, match=match):
            call()
    for t in (q, k, w, f):
        t.requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.qk_norm_rope(q, k, pos, f, w, w)
        with torch.no_grad():
            ops.qk_norm_rope(q, k, pos, f, w, w)
        t.requires_grad_(False)
    cache[1].requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.append_kv(k, v, *cache, table, pos)
