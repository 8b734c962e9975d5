"""Attention of one new token over a paged cache (`ops.paged_attention`) against its definition in 64 bits."""
import pytest
import torch

from tests.attention_util import DTYPES, attention64, check_attention, paged, rand

pytestmark = pytest.mark.gpu


def make(lengths, H, K, D, page, dtype, seed=0, order="pages", width=None, sharp=1.5):
    k = [rand(seed + 10 * s, n, K, D, dtype=dtype) for s, n in enumerate(lengths)]
    v = [rand(seed + 10 * s + 1, n, K, D, dtype=dtype) for s, n in enumerate(lengths)]
    q = rand(seed + 5, len(lengths), H, D, dtype=dtype, scale=sharp)
    return q, k, v, *paged(k, v, lengths, page, seed, order, width=width), torch.tensor(lengths, dtype=torch.int32, device="cuda")


def expected(q, k, v, window=None, scale=None):
    parts = [attention64(q[s:s + 1], k[s], v[s], torch.tensor([len(k[s]) - 1], device="cuda"), scale, window) for s in range(len(k))]
    return tuple(torch.cat([p[i] for p in parts]) for i in range(3))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,H,K,D,page,window", [
    ([1], 1, 1, 64, 8, None), ([1, 2, 15, 16, 17, 63, 64, 65], 8, 2, 128, 16, None), ([0, 5, 0, 300, 0], 4, 1, 64, 16, None), ([1000], 32, 8, 128, 16, None),
    ([257, 1, 4096, 33], 8, 8, 128, 64, None), ([500, 777], 40, 2, 64, 8, None), ([2000, 3], 71, 1, 64, 32, None), ([700, 90], 6, 3, 80, 16, None), ([1025, 64], 4, 2, 256, 128, None),
    ([350], 12, 4, 192, 16, None), ([300, 7], 3, 1, 8, 8, None), ([300, 7], 3, 3, 72, 8, None), ([1000, 30, 4000], 8, 2, 128, 16, 100), ([1000, 17], 8, 2, 64, 8, 1), ([5000, 200, 1], 16, 4, 128, 512, 1000),
    ([33] * 300, 4, 2, 64, 16, None), ([9000], 14, 2, 96, 32, None), ([1, 20000], 7, 1, 128, 16, None)])
def test_against_definition(lengths, H, K, D, page, window, dtype):
    from nanoquant_b200 import ops

    q, k, v, kc, vc, table, n = make(lengths, H, K, D, page, dtype)
    got = ops.paged_attention(q, kc, vc, table, n, window=window)
    assert got.shape == q.shape and got.is_contiguous()
    check_attention(got, expected(q, k, v, window))
    assert torch.equal(got, ops.paged_attention(q, kc, vc, table, n, window=window))          # the same order of sums


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page,width", [(8, 128), (16, 64), (512, 2), (1024, 1), (8, 129), (16, 65)])
def test_many_sequences_of_middling_length(page, width, D):
    """Tables of 1024 tokens for 128 key heads in all, which one launch takes, and of more, which two do."""
    from nanoquant_b200 import ops

    lengths = [1, 1024, 0, 513, 300, 1000, 16, 777] * 8
    q, k, v, kc, vc, table, n = make(lengths, 4, 2, D, page, torch.bfloat16, width=width)
    check_attention(ops.paged_attention(q, kc, vc, table, n), expected(q, k, v, None))
    check_attention(ops.paged_attention(q, kc, vc, table, n, window=301), expected(q, k, v, 301))


@pytest.mark.parametrize("lengths,H,K,D,page,width", [
    ([20, 0, 700] * 50, 32, 32, 64, 16, 130), ([1500, 3, 0, 900], 128, 128, 64, 16, None), ([300, 1, 64] * 20, 128, 128, 8, 16, 70), ([40, 1100, 7] * 45, 8, 4, 128, 32, 40),
    ([5, 2000, 0, 130] * 120, 2, 1, 64, 64, 64), ([1200, 80], 60, 20, 256, 16, None), ([700], 300, 150, 8, 8, 200), ([2100, 9] * 3, 200, 5, 128, 64, None)])
def test_more_sequences_or_heads_than_the_warps_take_at_once(lengths, H, K, D, page, width):
    """Key heads by which the warps do not divide, more of them than get groups of their own, more sequences than groups."""
    from nanoquant_b200 import ops

    q, k, v, kc, vc, table, n = make(lengths, H, K, D, page, torch.bfloat16, width=width)
    got = ops.paged_attention(q, kc, vc, table, n)
    check_attention(got, expected(q, k, v))
    assert torch.equal(got, ops.paged_attention(q, kc, vc, table, n))


@pytest.mark.parametrize("width", [None, 400])
def test_order_of_the_cache_and_width_of_the_table(width):
    """Heads outside the tokens of a page, keys and values in one tensor, rows of the table apart, a table far wider than the sequences: the same numbers within the bound (a wide
    table splits the sequences over the SMs)."""
    from nanoquant_b200 import ops

    lengths = [100, 9, 230]
    q, k, v, kc, vc, table, n = make(lengths, 8, 2, 64, 16, torch.bfloat16, order="heads", width=width)
    want = expected(q, k, v)
    check_attention(ops.paged_attention(q, kc, vc, table, n), want)
    both = torch.stack((kc, vc), 3)                               # [pages, page, K, 2, D]
    wide = torch.full((3, table.size(1) + 5), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, 2:-3] = table
    check_attention(ops.paged_attention(q.transpose(0, 1).contiguous().transpose(0, 1), both[..., 0, :], both[..., 1, :], wide[:, 2:-3], n), want)
    check_attention(ops.paged_attention(rand(1, 3, 8, 65, dtype=torch.bfloat16)[..., 1:].copy_(q), kc, vc, table, n), want)


@pytest.mark.parametrize("page", [8, 16, 128])
def test_what_is_not_seen_has_no_influence(page):
    """Rest of the last page, tokens and pages in front of a window, sequences of no tokens: NaN everywhere there, and places that do not exist in the table."""
    from nanoquant_b200 import ops

    lengths, window = [301, 40, 1000], 70
    q, k, v, kc, vc, table, n = make(lengths, 4, 2, 128, page, torch.float16)
    want = expected(q, k, v, window)
    for s, m in enumerate(lengths):
        for t in range(max(0, m - window)):
            p = table[s, t // page].item()
            kc[p, t % page] = float("nan")
            vc[p, t % page] = float("inf")
        table[s, :max(0, m - window) // page] = -1
    check_attention(ops.paged_attention(q, kc, vc, table, n, window=window), want)


@pytest.mark.parametrize("page,window", [(8, 70), (8, 3), (16, 33), (32, 40), (64, 64)])
def test_narrow_heads_and_pages_that_are_not_seen(page, window):
    """Heads of 64 columns, whose steps have several pages: those outside a window are NaN, or do not exist, one after the other in a step."""
    from nanoquant_b200 import ops

    lengths = [301, 40, 1000, 67, 0, 9]
    q, k, v, kc, vc, table, n = make(lengths, 8, 2, 64, page, torch.bfloat16)
    want = expected(q, k, v, window)
    for s, m in enumerate(lengths):
        for t in range(max(0, m - window)):
            p = table[s, t // page].item()
            kc[p, t % page] = float("nan")
            vc[p, t % page] = float("inf")
        table[s, :max(0, m - window) // page] = -1
    check_attention(ops.paged_attention(q, kc, vc, table, n, window=window), want)


@pytest.mark.parametrize("width", [16, 100])
def test_sequences_that_are_not_there_are_nan(width):
    """A page outside the cache, a length beyond the table: NaN in all of that sequence's outputs, the others untouched."""
    from nanoquant_b200 import ops

    lengths = [100, 200, 60, 16, 130]
    q, k, v, kc, vc, table, n = make(lengths, 8, 2, 64, 16, torch.bfloat16, width=width)
    o, avg, all_v = expected(q, k, v)
    table[1, 7] = kc.size(0)
    table[3, 0] = -1
    n[4] = 16 * width + 1
    got = ops.paged_attention(q, kc, vc, table, n)
    assert torch.isnan(got[[1, 3, 4]]).all()
    check_attention(got[[0, 2]], (o[[0, 2]], avg[[0, 2]], all_v[[0, 2]]))
    n[:] = torch.tensor([-5, 0, -2 ** 31, 0, 0], device="cuda")
    assert (ops.paged_attention(q, kc, vc, table, n) == 0).all()


def test_scores_of_any_size():
    """One score far above the others, large ones of both signs, a scale of the caller's; infinities as torch's softmax has them."""
    from nanoquant_b200 import ops

    q, k, v, kc, vc, table, n = make([600], 4, 1, 64, 16, torch.float16)
    q[0, 0] *= 20
    for scale in (None, 0.01, 1.0):
        # (scores of up to 2^9 instead of 2^6: an exponent's error is 2^-15 of it)
        o, avg, all_v = expected(q, k, v, scale=scale)
        got = ops.paged_attention(q, kc, vc, table, n, scale=scale)
        assert ((got.double() - o).abs() <= 2.0 ** -11 * o.abs() + (2.0 ** -10 + 2.0 ** -9) * avg + 2.0 ** -25 * (1 + all_v)).all()
    kc[table[0, 3].item(), 5, 0] = float("nan")
    assert torch.isnan(ops.paged_attention(q, kc, vc, table, n)).all()


def test_long_cache_with_64_bit_offsets():
    """Elements of the cache beyond 2^31, and more pages than the other tests have."""
    from nanoquant_b200 import ops

    pages, page, K, D = 40000, 64, 8, 128                         # 2.6e9 elements each
    kc, vc = (torch.zeros((pages, page, K, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    where = torch.tensor([pages - 1, 2, pages - 2, 33000], device="cuda")
    k, v = rand(0, 4 * page, K, D, dtype=torch.bfloat16), rand(1, 4 * page, K, D, dtype=torch.bfloat16)
    q = rand(2, 1, 32, D, dtype=torch.bfloat16)
    table, n = where.int()[None], torch.tensor([250], dtype=torch.int32, device="cuda")
    pos = torch.arange(256, device="cuda")
    ops.append_kv(k, v, kc, vc, table, pos, torch.zeros(256, dtype=torch.int32, device="cuda"))
    assert torch.equal(kc[where].view(-1, K, D), k) and torch.equal(vc[where].view(-1, K, D), v)
    want = attention64(q, k[:250], v[:250], torch.tensor([249], device="cuda"))
    check_attention(ops.paged_attention(q, kc, vc, table, n), want)
    check_attention(ops.prompt_attention(q, kc, vc, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), block_table=table, lengths=n), want)


def test_refusals():
    from nanoquant_b200 import ops

    q, k, v, kc, vc, table, n = make([30, 40], 8, 2, 64, 16, torch.float16)
    for match, call in (
            ("CUDA", lambda: ops.paged_attention(q.cpu(), kc, vc, table, n)), ("Half or BFloat16", lambda: ops.paged_attention(q.float(), kc, vc, table, n)), ("k_cache", lambda: ops.paged_attention(q.bfloat16(), kc, vc, table, n)),
            ("no multiple", lambda: ops.paged_attention(q[:, :7], kc, vc, table, n)), ("expected \\[sequences", lambda: ops.paged_attention(q[None], kc, vc, table, n)), ("lengths", lambda: ops.paged_attention(q, kc, vc, table, n.long())),
            ("lengths", lambda: ops.paged_attention(q, kc, vc, table, n[:1])), ("block_table", lambda: ops.paged_attention(q, kc, vc, table[:1], n)), ("block_table", lambda: ops.paged_attention(q, kc, vc, table[0], n)),
            ("v_cache", lambda: ops.paged_attention(q, kc, vc[:, :8], table, n)), ("power of two", lambda: ops.paged_attention(q, kc[:, :12], vc[:, :12], table, n)), ("k_cache has shape", lambda: ops.paged_attention(q, kc[..., :32], vc, table, n)),
            ("in place", lambda: ops.paged_attention(q, kc.flip(0)[..., ::2].repeat(1, 1, 1, 2)[..., ::1].transpose(2, 3).contiguous().transpose(2, 3), vc, table, n)), ("k_cache has shape", lambda: ops.paged_attention(q, kc[:0], vc[:0], table, n))):
        with pytest.raises(RuntimeError, match=match):
            call()
    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(window=0), dict(window=-3)):
        with pytest.raises(ValueError):
            ops.paged_attention(q, kc, vc, table, n, **kw)
    q.requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.paged_attention(q, kc, vc, table, n)


@pytest.mark.parametrize("width", [None, 1000])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scores_of_minus_infinity(D, width):
    """As torch's softmax has them: next to finite ones a weight of zero, and NaN where all of a query are so (which is not one that sees nothing); with a wide table by several CTAs."""
    from nanoquant_b200 import ops

    lengths, infinite = [250, 250, 1, 0, 130, 40], [250, 240, 1, 0, 0, 39]
    q, k, v, kc, vc, table, n = make(lengths, 4, 2, D, 16, torch.bfloat16, width=width)
    q[..., 0] = -1.0
    for s, m in enumerate(infinite):
        for t in range(m):
            kc[table[s, t // 16].item(), t % 16, :, 0] = float("inf")
    got = ops.paged_attention(q, kc, vc, table, n)
    assert torch.isnan(got[[0, 2]]).all() and (got[3] == 0).all()
    some = [1, 4, 5]
    check_attention(got[some], expected(q[some], [k[s][infinite[s]:] for s in some], [v[s][infinite[s]:] for s in some]))
    got = ops.paged_attention(q, kc, vc, table, n, window=11)
    assert torch.isnan(got[[0, 2]]).all() and (got[3] == 0).all() and not torch.isnan(got[some]).any()


@pytest.mark.parametrize("width", [None, 1000])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_small_weights(D, width):
    """fp16: one key 2^25.2 above all others, which by themselves make up the result.  A weight's subnormal half step is 2^-32 of the largest weight (they are formed 2^7 times as large)."""
    from nanoquant_b200 import ops

    lengths = [250, 17, 100]
    q, k, v, kc, vc, table, n = make(lengths, 4, 2, D, 16, torch.float16, width=width)
    q[:], q[..., 0] = 0.0, 1.0
    for s, m in enumerate(lengths):
        k[s][:], k[s][0, :, 0] = 0.0, 25.1875
        v[s].abs_()[0] = 0.0
        at = table[s, torch.arange(m, device="cuda") // 16].long(), torch.arange(m, device="cuda") % 16
        kc[at], vc[at] = k[s], v[s]
    scale = 0.69314718
    o, avg, all_v = expected(q, k, v, scale=scale)
    got = ops.paged_attention(q, kc, vc, table, n, scale=scale)
    bound = 2.0 ** -11 * o + (2.0 ** -10 + 2.0 ** -12) * avg + 2.0 ** -32 * all_v + 2.0 ** -25           # (the last: half a step of the result)
    assert ((got.double() - o).abs() <= bound * (1 + 2.0 ** -8)).all()
