"""Attention of packed prompts (`ops.prompt_attention`), over themselves, other keys or a paged cache, against its definition in 64 bits."""
import pytest
import torch

from tests.attention_util import DTYPES, attention64, check_attention, paged, rand

pytestmark = pytest.mark.gpu


def starts(lengths, first=0):
    return torch.tensor([first + sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device="cuda")


def expected(q, ks, vs, lengths, window=None, scale=None, causal=True, first=0):
    """Rows of no sequence: zeros."""
    out = [torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(3)]
    at = first
    for s, n in enumerate(lengths):
        place = torch.arange(n, device="cuda") + len(ks[s]) - n
        for o, part in zip(out, attention64(q[at:at + n], ks[s], vs[s], place, scale, window, causal)):
            o[at:at + n] = part
        at += n
    return out


def make(lengths, H, K, D, dtype, seed=0, sharp=1.5):
    T = sum(lengths)
    qkv = rand(seed, T, H + 2 * K, D)
    qkv[:, :H] *= sharp
    qkv = qkv.to(dtype)
    return qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:]


CASES = [([1], 1, 1, 64), ([128], 1, 1, 128), ([256], 2, 2, 128), ([257, 1, 127], 4, 1, 128), ([1, 2, 3, 37, 129, 300], 8, 2, 64), ([5, 0, 0, 70], 6, 3, 128), ([515], 14, 2, 64),
         ([300, 20], 71, 1, 64), ([200], 7, 1, 128), ([333, 64], 8, 8, 80), ([140, 3], 6, 2, 96), ([260, 65, 1], 4, 2, 256), ([130], 12, 4, 192), ([50, 9], 3, 1, 8), ([90], 100, 1, 24),
         ([1100, 900], 8, 2, 128), ([2049], 4, 4, 64), ([700], 2, 1, 256)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,H,K,D", CASES)
def test_against_definition(lengths, H, K, D, dtype):
    from nanoquant_b200 import ops

    q, k, v = make(lengths, H, K, D, dtype)
    cu = starts(lengths)
    ks, vs = k.split(lengths), v.split(lengths)
    got = ops.prompt_attention(q, k, v, cu)
    assert got.shape == q.shape and got.is_contiguous()
    check_attention(got, expected(q, ks, vs, lengths))
    assert torch.equal(got, ops.prompt_attention(q, k, v, cu))


@pytest.mark.parametrize("causal,window", [(False, None), (True, 1), (True, 100), (True, 513), (False, 64)])
@pytest.mark.parametrize("H,K,D", [(8, 2, 128), (2, 2, 64), (4, 1, 256)])
def test_masks(H, K, D, causal, window):
    from nanoquant_b200 import ops

    lengths = [700, 3, 130]
    q, k, v = make(lengths, H, K, D, torch.bfloat16)
    got = ops.prompt_attention(q, k, v, starts(lengths), causal=causal, window=window, scale=0.2)
    check_attention(got, expected(q, k.split(lengths), v.split(lengths), lengths, window, 0.2, causal))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_other_numbers_of_keys_than_queries(D, causal):
    """More keys: a prefix; fewer: rows that see nothing; none."""
    from nanoquant_b200 import ops

    lengths, keys = [130, 300, 20, 5, 260], [400, 100, 0, 6, 259]
    q = make(lengths, 4, 2, D, torch.float16)[0]
    k, v = make(keys, 4, 2, D, torch.float16, seed=1)[1:]
    got = ops.prompt_attention(q, k, v, starts(lengths), starts(keys), causal=causal)
    check_attention(got, expected(q, k.split(keys), v.split(keys), lengths, causal=causal))
    assert (got[430:450] == 0).all()
    if causal:
        assert (got[130:330] == 0).all() and (got[455] == 0).all()


def test_rows_of_no_sequence_are_zero():
    from nanoquant_b200 import ops

    lengths = [40, 300]
    q, k, v = make([7] + lengths + [1000], 4, 2, 128, torch.bfloat16)
    k[-1000:], v[-1000:], v[:7] = float("nan"), float("nan"), float("inf")
    spoil = torch.full((1347, 4, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    del spoil                                                      # (what the allocator is likely to hand out next)
    got = ops.prompt_attention(q, k, v, starts(lengths, 7))
    check_attention(got, expected(q, k[7:347].split(lengths), v[7:347].split(lengths), lengths, first=7))
    assert (got[:7] == 0).all() and (got[347:] == 0).all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_neighbours_have_no_influence(D):
    """NaN and infinities in the sequences beside one, in the rows of the same step."""
    from nanoquant_b200 import ops

    lengths = [30, 100, 77]
    q, k, v = make(lengths, 4, 2, D, torch.float16)
    want = [t[30:130] for t in expected(q, k.split(lengths), v.split(lengths), lengths)]
    for t in (q, k, v):
        t[:30], t[130:] = float("nan"), float("inf")
    check_attention(ops.prompt_attention(q, k, v, starts(lengths))[30:130], want)


def piece(new, total, H, K, D, page, dtype, seed=0, order="pages"):
    k = [rand(seed + 10 * s, n, K, D, dtype=dtype) for s, n in enumerate(total)]
    v = [rand(seed + 10 * s + 1, n, K, D, dtype=dtype) for s, n in enumerate(total)]
    q = rand(seed + 3, sum(new), H, D, dtype=dtype, scale=1.5)
    kc, vc, table = paged(k, v, total, page, seed, order)
    return q, k, v, kc, vc, table, torch.tensor(total, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,total,H,K,D,page,window", [
    ([1], [1], 1, 1, 64, 16, None), ([100, 1, 30], [100, 500, 31], 8, 2, 128, 16, None), ([64], [1000], 4, 4, 64, 8, None), ([300, 2], [900, 130], 8, 2, 128, 128, None), ([70], [333], 4, 1, 80, 32, None),
    ([33, 0, 5], [97, 40, 5], 4, 2, 256, 16, None), ([200], [700], 4, 2, 128, 1024, None), ([150, 4], [800, 300], 8, 2, 128, 16, 100), ([9], [600], 2, 1, 64, 64, 50), ([40], [300], 2, 1, 256, 128, 70),
    ([12], [5], 4, 2, 128, 16, None), ([17], [0], 4, 2, 64, 16, None)])
def test_paged(new, total, H, K, D, page, window, dtype):
    """A piece of a prompt behind what the cache holds; everything that no query sees is NaN, and places in the table that are not needed do not exist."""
    from nanoquant_b200 import ops

    q, k, v, kc, vc, table, n = piece(new, total, H, K, D, page, dtype, order="heads" if page == 16 else "pages")
    want = expected(q, k, v, new, window)
    if window:
        for s, m in enumerate(total):                             # pages wholly in front of the first query's window
            table[s, :max(0, m - new[s] + 1 - window) // page] = -1
    check_attention(ops.prompt_attention(q, kc, vc, starts(new), block_table=table, lengths=n, window=window), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,total,H,K,D,page,window", [
    ([1], [3001], 8, 2, 128, 16, None), ([16, 2, 0], [5000, 100, 2000], 4, 2, 64, 32, None), ([70, 200, 3], [4000, 900, 33], 8, 1, 128, 64, None), ([5, 9], [2500, 2600], 4, 2, 256, 16, None),
    ([100], [9000], 6, 2, 80, 128, 2500), ([130], [2048], 14, 2, 96, 8, None)])
def test_few_tokens_behind_a_long_cache(new, total, H, K, D, page, window, dtype):
    """The keys of a block go to several CTAs, whose sums a second launch joins: parts that a tile or a row sees nothing of among them."""
    import ctypes

    from nanoquant_b200 import _lib, ops

    q, k, v, kc, vc, table, n = piece(new, total, H, K, D, page, dtype)
    d = _lib.AttentionDesc(q=1 << 16, k=1 << 16, v=1 << 16, out=1 << 16, cu_seqlens=1 << 16, lengths=1 << 16, block_table=1 << 16, k_slot=8, v_slot=8, table_stride=1, pages=kc.size(0),
                           max_pages=table.size(1), page_size=page, T=len(q), seqs=len(new), q_heads=H, k_heads=K, D=D, causal=1, scale=1.0)
    assert _lib.lib().nq_prompt_attention_scratch_bytes(ctypes.byref(d)) > 0
    want = expected(q, k, v, new, window)
    got = ops.prompt_attention(q, kc, vc, starts(new), block_table=table, lengths=n, window=window)
    check_attention(got, want)
    assert torch.equal(got, ops.prompt_attention(q, kc, vc, starts(new), block_table=table, lengths=n, window=window))
    packed = ops.prompt_attention(q, torch.cat(k), torch.cat(v), starts(new), starts(total), window=window)
    check_attention(packed, want)
    if total[0] < 5000:                                           # a page outside the cache: NaN, wherever the part is that has it
        table[0, total[0] // page // 2] = -1
        bad = ops.prompt_attention(q, kc, vc, starts(new), block_table=table, lengths=n, window=window)
        assert torch.isnan(bad[:new[0]]).all()
        check_attention(bad[new[0]:], [t[new[0]:] for t in want])


@pytest.mark.parametrize("D", [64, 256])
def test_sequences_that_are_not_there_are_nan(D):
    from nanoquant_b200 import ops

    new, total = [10, 200, 3, 40], [100, 300, 60, 64]
    q, k, v, kc, vc, table, n = piece(new, total, 4, 2, D, 16, torch.bfloat16)
    want = expected(q, k, v, new)
    table[1, 3] = kc.size(0)
    n[2] = 16 * table.size(1) + 1
    got = ops.prompt_attention(q, kc, vc, starts(new), block_table=table, lengths=n)
    assert torch.isnan(got[10:213]).all()
    rows = torch.cat((torch.arange(10), torch.arange(213, 253))).cuda()
    check_attention(got[rows], [t[rows] for t in want])


def test_maximum_that_keeps_growing():
    """Scores that grow along the sequence by more than the maximum may lag, step after step, and ones that fall."""
    from nanoquant_b200 import ops

    n, H, D = 1500, 2, 128
    for sign in (1, -1):
        q, k, v = make([n], H, H, D, torch.float16)
        q, k = q.clone(), k.clone()
        q[..., 0] = 16.0
        k[..., 0] = sign * torch.arange(n, device="cuda")[:, None] * (3.0 / 64)      # products to 2^10.2, scaled below 2^6.7
        want = expected(q, [k], [v], [n])
        o, avg, all_v = want
        got = ops.prompt_attention(q, k, v, starts([n]))
        assert ((got.double() - o).abs() <= 2.0 ** -11 * o.abs() + (2.0 ** -10 + 2.0 ** -11) * avg + 2.0 ** -25 * (1 + all_v)).all()


def test_more_sequences_than_a_warp():
    from nanoquant_b200 import ops

    lengths = [(7 * i) % 23 for i in range(150)]
    q, k, v = make(lengths, 4, 2, 64, torch.bfloat16)
    check_attention(ops.prompt_attention(q, k, v, starts(lengths)), expected(q, k.split(lengths), v.split(lengths), lengths))


def test_layouts():
    from nanoquant_b200 import ops

    lengths = [100, 60]
    q, k, v = make(lengths, 4, 2, 64, torch.float16)
    want = ops.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), starts(lengths))
    odd = rand(0, 160, 4, 65, dtype=torch.float16)[..., 1:]
    odd[:, :4] = q
    wide = starts(lengths).repeat_interleave(2)[::2]
    for a, b, c in ((odd, k, v), (q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(0, 1).contiguous().transpose(0, 1), v), (q, k.permute(2, 0, 1).contiguous().permute(1, 2, 0), v)):
        assert torch.equal(ops.prompt_attention(a, b, c, wide), want)
    same = ops.prompt_attention(q, k[:, :1].expand(160, 4, 64), v[:, :1].expand(160, 4, 64), starts(lengths))
    # (a row's sums do not depend on the heads beside it)
    assert torch.equal(same, ops.prompt_attention(q, k[:, :1].repeat(1, 4, 1), v[:, :1].repeat(1, 4, 1), starts(lengths)))
    assert ops.prompt_attention(q[:0], k, v, starts([0])).shape == (0, 4, 64)


def test_refusals():
    from nanoquant_b200 import ops

    lengths = [30, 40]
    q, k, v = make(lengths, 8, 2, 64, torch.float16)
    cu = starts(lengths)
    kc, vc, table = paged(k.split(lengths), v.split(lengths), lengths, 16)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for match, call in (
            ("CUDA", lambda: ops.prompt_attention(q.cpu(), k, v, cu)), ("Half or BFloat16", lambda: ops.prompt_attention(q.float(), k, v, cu)), ("k is", lambda: ops.prompt_attention(q, k.bfloat16(), v, cu)),
            ("v has shape", lambda: ops.prompt_attention(q, k, v[:-1], cu)), ("no multiple", lambda: ops.prompt_attention(q[:, :7], k, v, cu)), ("expected \\[tokens", lambda: ops.prompt_attention(q[None], k, v, cu)),
            ("cu_seqlens", lambda: ops.prompt_attention(q, k, v, cu.long())), ("cu_seqlens", lambda: ops.prompt_attention(q, k, v, cu[:1])), ("cu_seqlens", lambda: ops.prompt_attention(q, k, v, None)),
            ("cu_seqlens_k", lambda: ops.prompt_attention(q, k, v, cu, cu[:2])), ("go together", lambda: ops.prompt_attention(q, kc, vc, cu, block_table=table)), ("go together", lambda: ops.prompt_attention(q, k, v, cu, lengths=n)),
            ("cu_seqlens_k", lambda: ops.prompt_attention(q, kc, vc, cu, cu, table, n)), ("lengths", lambda: ops.prompt_attention(q, kc, vc, cu, block_table=table, lengths=n[:1])),
            ("block_table", lambda: ops.prompt_attention(q, kc, vc, cu, block_table=table[:1], lengths=n)), ("k has shape", lambda: ops.prompt_attention(q, k[:0], v[:0], cu)),
            ("128", lambda: ops.prompt_attention(rand(0, 4, 130, 64, dtype=torch.float16), k[:4, :1], v[:4, :1], cu)), ("expected \\[pages", lambda: ops.prompt_attention(q, k, v, cu, block_table=table, lengths=n))):
        with pytest.raises(RuntimeError, match=match):
            call()
    for kw in (dict(scale=0.0), dict(scale=float("inf")), dict(window=0)):
        with pytest.raises(ValueError):
            ops.prompt_attention(q, k, v, cu, **kw)
    k.requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.prompt_attention(q, k, v, cu)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new,total,page,window", [
    ([3, 1, 20], [300, 77, 500], 16, 70), ([5], [131], 128, 40), ([2, 300], [1000, 900], 1024, 100), ([1], [4001], 64, 3500), ([1, 2, 1, 1], [130, 131, 200, 90], 8, 3)])
def test_what_no_query_sees_has_no_influence(new, total, page, window, D):
    """Tokens ahead of the first query's window that were never stored, in pages that do not exist or that it shares with others: keys NaN, values NaN or infinite."""
    from nanoquant_b200 import ops

    q, k, v, kc, vc, table, n = piece(new, total, 4, 2, D, page, torch.bfloat16)
    want = expected(q, k, v, new, window=window)
    for s, (m, t) in enumerate(zip(new, total)):
        unseen = max(0, t - m + 1 - window)
        for i in range(unseen):
            p = table[s, i // page].item()
            kc[p, i % page], vc[p, i % page] = float("nan"), float("inf") if i % 2 else float("nan")
        table[s, :unseen // page] = -1
    check_attention(ops.prompt_attention(q, kc, vc, starts(new), block_table=table, lengths=n, window=window), want)
    for x, y, m, t in zip(k, v, new, total):
        x[:max(0, t - m + 1 - window)], y[:max(0, t - m + 1 - window)] = float("nan"), float("nan")
    check_attention(ops.prompt_attention(q, torch.cat(k), torch.cat(v), starts(new), starts(total), window=window), want)



@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("where", ["step", "last"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_maximum_left_behind_in_a_step_without_masks(D, where, dtype):
    """Scores that rise by 2^16 with every step of keys, or in a step's last 32 keys: weights that were formed with the maximum before are formed, and stored, once more."""
    from nanoquant_b200 import ops

    n, step = 520, 128 if D <= 128 else 64
    q, k, v = (rand(i, n, 2, D, scale=s).to(dtype) for i, s in ((0, 0.1), (1, 1.0), (2, 1.0)))
    at = torch.arange(n, device="cuda")
    q[..., 0] = 16.0
    k[..., 0] = (at // step + (at % step >= step - 32) * (where == "last"))[:, None].to(dtype)
    scale = 0.69314718                                            # 16 powers of two a step, 2^7.2 at most: natural exponents below 2^6.7
    o, avg, all_v = expected(q, [k], [v], [n], scale=scale)
    # (as check_attention has it, with scores of up to 2^6.7: up to 16 products of 16 columns, each cut off at 2^-23 of them, are 2^-12.3 of a weight, and as much of the sum)
    u = torch.finfo(dtype).eps / 2
    for causal in (True, False):
        want = (o, avg, all_v) if causal else expected(q, [k], [v], [n], scale=scale, causal=False)
        got = ops.prompt_attention(q, k, v, starts([n]), causal=causal, scale=scale)
        bound = u * want[0].abs() + (2 * u + 2.0 ** -11) * want[1] + (2.0 ** -25 if dtype == torch.float16 else 0.0) * (1 + want[2])
        assert ((got.double() - want[0]).abs() <= bound * (1 + 2.0 ** -8)).all()
        assert torch.equal(got, ops.prompt_attention(q, k, v, starts([n]), causal=causal, scale=scale))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new,total,page,window", [
    ([400, 30], [500, 30], 16, None), ([300, 5], [300, 900], 8, None), ([40, 3], [60, 70], 64, None), ([700, 9], [900, 40], 32, 100), ([20, 1], [6000, 300], 16, None), ([30], [4000], 8, 3000),
    ([300, 7], [40, 7], 16, None), ([600] + [8] * 300, [600] + [40] * 300, 16, None)])
def test_a_page_that_is_not_there_makes_its_whole_sequence_nan(new, total, page, window, D):
    """The first and the last page that some query of the sequence sees, one that only a few of them do: NaN in all of its outputs, those ahead of the page and those that see nothing among
    them, in every run; the other sequences are as without it.  Pages ahead of every window are not looked at."""
    from nanoquant_b200 import ops

    q, k, v, kc, vc, table, n = piece(new, total, 4, 2, D, page, torch.bfloat16)
    cu = starts(new)
    fine = ops.prompt_attention(q, kc, vc, cu, block_table=table, lengths=n, window=window)
    check_attention(fine, expected(q, k, v, new, window))
    first = max(0, total[0] - new[0] + 1 - window) // page if window else 0
    last = (total[0] - 1) // page
    for at in sorted({first, (first + last) // 2, last}):
        for wrong in (-1, kc.size(0), 2 ** 31 - 1):
            bad = table.clone()
            bad[0, at] = wrong
            bad[0, :first] = wrong                                # (nobody sees those)
            for _ in range(3):
                got = ops.prompt_attention(q, kc, vc, cu, block_table=bad, lengths=n, window=window)
                assert torch.isnan(got[:new[0]]).all(), (at, wrong)
                assert torch.equal(got[new[0]:], fine[new[0]:])
    bad = table.clone()
    bad[0, :first] = -1
    bad[0, last + 1:] = kc.size(0)                                # (nor what lies behind the last token)
    assert torch.equal(ops.prompt_attention(q, kc, vc, cu, block_table=bad, lengths=n, window=window), fine)


@pytest.mark.parametrize("behind", [0, 300, 3000])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scores_of_minus_infinity(D, behind):
    """As torch's softmax has them: next to finite ones a weight of zero, and NaN for a query whose scores are all so (which is not one that sees nothing)."""
    from nanoquant_b200 import ops

    new, first = (200, 130) if not behind else (20, behind + 7)
    total = new + behind
    q, k, v, kc, vc, table, n = piece([new], [total], 4, 2, D, 16, torch.bfloat16)
    place = torch.arange(new, device="cuda") + behind
    q[..., 0] = -1.0
    k[0][:first, :, 0] = float("inf")
    kc[table[0].long()] = torch.cat((k[0], k[0].new_zeros(table.size(1) * 16 - total, 2, D))).view(-1, 16, 2, D)
    some = place >= first
    want = attention64(q[some], k[0][first:], v[0][first:], place[some] - first)
    cu = starts([new])
    for got in (ops.prompt_attention(q, kc, vc, cu, block_table=table, lengths=n), ops.prompt_attention(q, k[0], v[0], cu, starts([total]))):
        assert torch.isnan(got[~some]).all()
        check_attention(got[some], want)
    got = ops.prompt_attention(q, kc, vc, cu, block_table=table, lengths=n, window=2)
    assert torch.isnan(got[~some]).all() and not torch.isnan(got[some]).any()
    k[0][..., 0] = float("inf")
    kc[table[0].long(), ..., 0] = float("inf")
    for causal in (True, False):
        assert torch.isnan(ops.prompt_attention(q, kc, vc, cu, block_table=table, lengths=n, causal=causal)).all()
        assert torch.isnan(ops.prompt_attention(q, k[0], v[0], cu, starts([total]), causal=causal)).all()
    assert (ops.prompt_attention(q, kc, vc, cu, block_table=table, lengths=torch.zeros_like(n)) == 0).all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_small_weights(D):
    """fp16: one key 2^25.2 above all others, which by themselves make up the result.  A weight's subnormal half step is 2^-28 of the largest weight (they are formed 2^3 times as large)."""
    from nanoquant_b200 import ops

    n = 1000
    q, k, v = (torch.zeros((n, 2, D), dtype=torch.float16, device="cuda") for _ in range(3))
    q[..., 0], k[0, :, 0], v[1:] = 1.0, 25.1875, rand(0, n - 1, 2, D).abs().half()
    scale = 0.69314718
    cu = starts([n])
    o, avg, all_v = expected(q, [k], [v], [n], scale=scale)
    got = ops.prompt_attention(q, k, v, cu, scale=scale)
    bound = 2.0 ** -11 * o + (2.0 ** -10 + 2.0 ** -12) * avg + 2.0 ** -28 * all_v + 2.0 ** -25           # (the last: half a step of the result)
    assert ((got.double() - o).abs() <= bound * (1 + 2.0 ** -8)).all()
    check_attention(ops.prompt_attention(q, k, v, cu, scale=scale, causal=False), expected(q, [k], [v], [n], scale=scale, causal=False))


def parts_of(q, kc, table, seqs, K):
    """Scratch of a call over the cache: none where no block is cut."""
    import ctypes

    from nanoquant_b200 import _lib

    d = _lib.AttentionDesc(q=1 << 16, k=1 << 16, v=1 << 16, out=1 << 16, cu_seqlens=1 << 16, lengths=1 << 16, block_table=1 << 16, k_slot=8, v_slot=8, table_stride=1, pages=kc.size(0),
                           max_pages=table.size(1), page_size=kc.size(1), T=len(q), seqs=seqs, q_heads=q.size(1), k_heads=K, D=q.size(2), causal=1, scale=1.0)
    return _lib.lib().nq_prompt_attention_scratch_bytes(ctypes.byref(d))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,total,H,K,D,page,window", [
    ([40, 3, 1], [2000, 2, 700], 8, 2, 128, 16, None), ([300, 5], [100, 90], 4, 2, 64, 16, None), ([200, 2], [900, 4000], 4, 1, 256, 64, None), ([30, 30], [1500, 3], 4, 2, 96, 8, 300),
    ([600], [600], 8, 2, 64, 32, None)])
def test_tables_far_wider_than_the_sequences(new, total, H, K, D, page, window, causal):
    """A table for 65536 tokens, by whose width blocks are cut: lengths that give many parts, one, or none; fewer keys than queries; every query over all keys (as over another text's)."""
    from nanoquant_b200 import ops

    q, k, v, kc, vc, table, n = piece(new, total, H, K, D, page, torch.bfloat16)
    wide = torch.full((len(new), 65536 // page), -9, dtype=torch.int32, device="cuda")
    wide[:, :table.size(1)] = table
    assert parts_of(q, kc, wide, len(new), K) > 0
    want = expected(q, k, v, new, window, causal=causal)
    got = ops.prompt_attention(q, kc, vc, starts(new), block_table=wide, lengths=n, causal=causal, window=window)
    check_attention(got, want)
    assert torch.equal(got, ops.prompt_attention(q, kc, vc, starts(new), block_table=wide, lengths=n, causal=causal, window=window))
    check_attention(ops.prompt_attention(q, kc, vc, starts(new), block_table=table, lengths=n, causal=causal, window=window), want)


def test_few_queries_over_all_keys_of_another_text():
    """Packed keys, no causal order, blocks cut along the keys."""
    from nanoquant_b200 import ops

    new, total = [9, 70, 1], [5000, 2000, 3000]
    q = make(new, 8, 2, 128, torch.float16)[0]
    k, v = make(total, 8, 2, 128, torch.float16, seed=1)[1:]
    got = ops.prompt_attention(q, k, v, starts(new), starts(total), causal=False)
    check_attention(got, expected(q, k.split(total), v.split(total), new, causal=False))
