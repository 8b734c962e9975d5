"""Cross entropy over the head without the logits (`ops.linear_cross_entropy`) against its definition in 64 bits.

Bounds, from magnitudes S[t, v] = sum_k |h[t, k] w[v, k]|.  A logit is a sum over N / 16 matrix instructions, each of which may cut the sum off at
2^-23 of it (and so may the few additions of partial sums): at most E = (N / 16 + 16) 2^-23 max_v S.  lse moves by no more than the logits do; the exponentials,
their sum and the logarithm add 2^-19 of (1 + |lse|) at most.

Gradients: d = g (p - [target]) has the relative error 2 E + 2^-18 of p and is rounded to the type, half a step u (fp16 after scaling by 2^14 / max|g|, where
numbers below 2^-14 are off by 2^-25 at most); a sum of n products adds (n / 16 + 16) 2^-23 of their magnitudes; the result is rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
DTYPES = [torch.float16, torch.bfloat16]


def make(T, N, V, dtype, seed=0, ignored=0.25, wide=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")
    w = (rand(V, N) * (1.28 / N ** 0.5)).to(dtype)
    t = torch.randint(V, (T,), generator=g, device="cuda")
    h = (rand(T, N) + 8 * torch.rand((T, 1), generator=g, device="cuda") * w[t].float()).to(dtype)
    t[torch.rand(T, generator=g, device="cuda") < ignored] = -100
    t[0] = V - 1
    return h, w, t if wide else t.int()


def reference(h, w, t, reduction, g, ignore=-100):
    """(loss, bound), (dh, bound), (dw, bound)"""
    dtype, u = h.dtype, torch.finfo(h.dtype).eps / 2
    h, w, t = h.detach().double(), w.detach().double(), t.long()
    T, N, V = *h.shape, w.size(0)
    live = t != ignore
    at = torch.where(live, t, 0)[:, None]
    l = h @ w.T
    E = (N / 16 + 16) * 2.0 ** -23 * (h.abs() @ w.abs().T).amax(1)
    lse = torch.logsumexp(l, 1)
    zero = torch.zeros_like(lse)
    each = torch.where(live, lse - l.gather(1, at)[:, 0], zero)
    each_b = torch.where(live, 2 * E + 2.0 ** -19 * (1 + lse.abs()), zero)
    count = live.sum()
    g = torch.as_tensor(g, device=h.device).double().expand(T)
    if reduction == "none":
        loss, loss_b = each, each_b + 2.0 ** -23 * each.abs()
    else:
        k = 1 if reduction == "sum" else count
        loss, loss_b = each.sum() / k, each_b.sum() / k + 2.0 ** -23 * each.abs().sum() / k
        g = g / k
    g = torch.where(live, g, zero)
    p = (l - lse[:, None]).exp()
    d = p.clone()
    d.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    d, p = d * g[:, None], p * g[:, None].abs()
    off = p * (2 * E + 2.0 ** -18)[:, None] + d.abs() * u + (2.0 ** -25 / 2 ** 14 * g.abs().max() if dtype == torch.float16 else 0)
    n = lambda k: (k / 16 + 64) * 2.0 ** -23
    dh, dw = d @ w, d.T @ h
    dh_b = off @ w.abs() + n(V) * (d.abs() @ w.abs()) + u * dh.abs() + TINY[dtype]
    dw_b = off.T @ h.abs() + n(T) * (d.abs().T @ h.abs()) + u * dw.abs() + TINY[dtype]
    return (loss, loss_b), (dh, dh_b), (dw, dw_b)


def check(got, want):
    for name, x, (x64, bound) in zip(("loss", "dh", "dw"), got, want):
        assert x.shape == x64.shape and torch.isfinite(x).all(), name
        excess = ((x.double() - x64).abs() - bound * (1 + 2.0 ** -9)).max().item()
        assert excess <= 0, (name, excess)


def run(h, w, t, reduction="mean", g=None, **kw):
    from nanoquant_b200 import ops

    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = ops.linear_cross_entropy(h, w, t, reduction=reduction, **kw)
    g = torch.ones_like(loss) if g is None else torch.as_tensor(g, dtype=torch.float32, device="cuda").expand(loss.shape)
    return [loss.detach(), *torch.autograd.grad(loss, (h, w), g)]


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,V", [
    (1, 8, 1), (1, 64, 2), (2, 128, 15), (5, 72, 300), (31, 256, 1000), (77, 512, 1003), (128, 200, 4097), (129, 256, 999), (255, 64, 130),
    (257, 1024, 2050), (300, 4096, 500), (640, 136, 33333)])
def test_loss_and_gradients_match_definition(T, N, V, dtype, reduction):
    h, w, t = make(T, N, V, dtype, seed=T + V, wide=V % 2 == 0)
    # (fp16 as in training: a scaled loss, without which the gradients of a mean are below the smallest numbers)
    g = (torch.rand(T, device="cuda") - 0.3) * 64 if reduction == "none" else 64.0
    check(run(h, w, t, reduction, g), reference(h, w, t, reduction, g))


@pytest.mark.parametrize("dtype", DTYPES)
def test_loss_in_several_pieces_of_the_vocabulary(dtype):
    """More tokens times words than the scratch holds at once, a last piece that is shorter."""
    T, N, V = 2100, 64, 130001
    h, w, t = make(T, N, V, dtype, seed=3)
    got, rows = run(h, w, t, "sum", 4.0), slice(0, 50)
    want = reference(h[rows], w, t[rows], "none", 4.0)      # (the whole in 64 bits takes too long: some tokens, then the sum of all of dw's columns)
    check([torch.nn.functional.pad(got[1][rows], (0, 0))], [want[1]])
    lw = torch.logsumexp(h.double() @ w.double().T, 1)
    live = t != -100
    d = (h.double() @ w[-3000:].double().T - lw[:, None]).exp()
    hit = t - (V - 3000)
    inside = live & (hit >= 0)
    d[inside, hit[inside]] -= 1
    d *= 4.0 * live[:, None]
    dw = d.T @ h.double()
    u = torch.finfo(dtype).eps / 2
    E = (N / 16 + 16) * 2.0 ** -23 * (h.double().abs() @ w.double().abs().T).amax()
    bound = (u + 2 * E + 2.0 ** -17) * (d.abs().T @ h.double().abs()) + u * dw.abs() + 2.0 ** -16
    assert ((got[2][-3000:].double() - dw).abs() <= bound).all()


@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_more_tokens_than_one_product_takes(reduction):
    """Several products of tokens, the last one of another kind; a token's loss is that of its own product alone."""
    from nanoquant_b200 import ops

    for T in (16384 + 100, 2 * 16384 + 300):
        h, w, t = make(T, 64, 700, torch.bfloat16, seed=T)
        got = run(h, w, t, reduction, 8.0)
        check(got, reference(h, w, t, reduction, 8.0))
        if reduction == "none":
            for rows in (slice(0, 16384), slice(T // 16384 * 16384, T)):
                assert torch.equal(got[0][rows], ops.linear_cross_entropy(h[rows], w, t[rows], reduction="none"))


def test_gradient_matches_differences():
    """<dh, a> and <dw, b> against differences of the loss, with steps that the type holds exactly."""
    from nanoquant_b200 import ops

    T, N, V = 20, 256, 700
    h, w, t = make(T, N, V, torch.float16, seed=21)
    h, w = (h * 64).round() / 64, (w * 1024).round() / 1024
    sign = lambda x: (torch.randint(0, 2, x.shape, device="cuda") * 2 - 1).half()
    _, dh, dw = run(h, w, t, "sum", 1.0)
    f = lambda a, b: ops.linear_cross_entropy(a, b, t, reduction="none").double().sum().item()
    for x, d, step, call in ((h, dh, 2.0 ** -6, lambda v: f(h + v, w)), (w, dw, 2.0 ** -10, lambda v: f(h, w + v))):
        v = sign(x) * step
        slope, diff = (d.double() * v.double()).sum().item(), (call(v) - call(-v)) / 2
        # the gradients' own rounding, the two losses' errors, and the third-order term: the logits move by z, |f'''| z^3 / 6 < |z|^3 / 2
        z = ((v.double() @ w.double().T).abs().amax(1) if x is h else (h.double() @ v.double().T).abs().amax(1))
        bound = 2 * 2.0 ** -11 * (d.double() * v.double()).norm().item() * 4 + T * 1e-4 + (z ** 3).sum().item() / 2
        assert abs(slope - diff) <= bound and bound < 0.5 * abs(slope) + 1, (slope, diff, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,V,ignored", [(600, 1024, 200000, 0.5), (1030, 1024, 110000, 0.97), (2500, 2048, 20000, 0.1), (700, 2048, 80000, 0.0), (513, 2048, 100000, 1.0),
                                           (20000, 128, 40000, 0.3)])
def test_tokens_without_a_target_take_no_part(T, N, V, ignored, dtype):
    """Sizes at which the rows that have a target are packed: a few, most, all and none of them (and one that is no word)."""
    h, w, t = make(T, N, V, dtype, seed=T, ignored=ignored)
    if ignored == 1.0:
        t[:] = -100
    else:
        t[7:200] = -100                      # whole runs, the last row among them
        t[-1] = -100
        t[3], t[250] = 5, V // 2
    if ignored == 0.0:
        t[t == -100] = 1
    live = t != -100
    clean = h.clone()
    h[~live] = float("nan")
    g = torch.rand(T, device="cuda") * 16
    got = run(h, w, t, "none", g)
    assert not got[1][~live].any() and not got[0][~live].any()
    rows = torch.cat([live.nonzero()[:40, 0], live.nonzero()[-40:, 0]])
    if len(rows):
        # 64 bits for some tokens, and for dw the words that are some tokens' targets and others
        want = reference(clean[rows], w, t[rows], "none", g[rows])
        u = torch.finfo(dtype).eps / 2
        for name, x, (x64, bound) in zip(("loss", "dh"), got, want):
            # (fp16: rounded relative to the largest |g| of all tokens)
            extra = 2.0 ** -25 / 2 ** 14 * 16 * w.double().abs().sum(0) if name == "dh" and dtype == torch.float16 else 0
            assert ((x[rows].double() - x64).abs() <= bound * (1 + 2.0 ** -9) + extra).all(), name
        words = torch.cat([t[rows], torch.arange(64, device="cuda")])
        hl, wl = clean[live].double(), w.double()
        lse = torch.cat([torch.logsumexp(c.double() @ wl.T, 1) for c in clean[live].split(256)])
        l = hl @ wl[words].T
        d = ((l - lse[:, None]).exp() - (t[live][:, None] == words).double()) * g[live].double()[:, None]
        E = (N / 16 + 16) * 2.0 ** -23 * (hl.abs() @ wl[words].abs().T)
        dw = d.T @ hl
        off = (d + (t[live][:, None] == words) * g[live][:, None]) * (2 * E + 2.0 ** -18 + 2 * E.amax(1, keepdim=True)) + d.abs() * u + 2.0 ** -25 / 2 ** 14 * 16
        bound = off.T @ hl.abs() + (T / 16 + 64) * 2.0 ** -23 * (d.abs().T @ hl.abs()) + u * dw.abs() + TINY[dtype]
        assert ((got[2][words].double() - dw).abs() <= bound * (1 + 2.0 ** -9)).all()
    else:
        assert not got[2].any()
    # invalid targets among them
    if len(rows):
        t[rows[0]] = V
        bad = run(h, w, t, "none", g)
        assert torch.isnan(bad[0][rows[0]]) and torch.isnan(bad[1][rows[0]]).all()
        others = torch.ones(T, dtype=torch.bool, device="cuda")
        others[rows[0]] = False
        assert torch.equal(bad[0][others], got[0][others]) and torch.equal(bad[1][others], got[1][others])
    # the packed rows of one call are those of the tokens alone
    if live.any() and ignored > 0:
        alone = run(clean[live], w, t[live].clamp(max=V - 1), "sum", 2.0)
        t2 = t.clamp(max=V - 1)
        both = run(h, w, t2, "sum", 2.0)
        assert abs(both[0] - alone[0]) <= 1e-5 * alone[0].abs() and ((both[1][live].double() - alone[1].double()).abs() <= 2.0 ** -7 * alone[1].double().abs() + 1e-4).all()


def test_packed_call_replayed_with_other_targets():
    """How many rows are packed is the device's knowledge: a captured step follows its targets, from none to all of the tokens."""
    from nanoquant_b200 import ops

    T, N, V = 1200, 1024, 90000
    h, w, t = make(T, N, V, torch.bfloat16, seed=31, ignored=0.0)
    h.requires_grad_(), w.requires_grad_()
    held = t.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.linear_cross_entropy(h, w, held, reduction="sum"), (h, w))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss = ops.linear_cross_entropy(h, w, held, reduction="sum")
            grads = torch.autograd.grad(loss, (h, w))
    torch.cuda.current_stream().wait_stream(side)
    for ignored in (0.4, 0.0, 1.0, 0.99, 0.05):
        with torch.no_grad():
            held.copy_(torch.where(torch.rand(T, device="cuda") < ignored, -100, t))
        graph.replay()
        want = ops.linear_cross_entropy(h, w, held, reduction="sum")
        for a, b in zip((loss, *grads), (want, *torch.autograd.grad(want, (h, w)))):
            assert torch.equal(a, b), ignored


def test_ignored_tokens_hold_anything():
    h, w, t = make(140, 64, 500, torch.bfloat16, seed=5, ignored=0.0)
    t[3::7] = 7
    want = run(h[t != 7], w, t[t != 7], "mean", ignore_index=7)
    h[3], h[10, 5], h[17] = float("nan"), float("inf"), 3e38
    loss, dh, dw = run(h, w, t, "mean", ignore_index=7)
    live = t != 7
    assert not dh[~live].any()
    u = 2.0 ** -8
    # the same tokens in other tiles: the same sums in another order
    assert abs(loss - want[0]) <= 1e-5 * want[0]
    assert ((dh[live].double() - want[1].double()).abs() <= 2 * u * want[1].double().abs() + 1e-4 * want[1].abs().max()).all()
    assert ((dw.double() - want[2].double()).abs() <= 2 * u * want[2].double().abs() + 1e-4 * want[2].abs().max()).all()


def test_no_target_at_all():
    h, w, _ = make(9, 64, 100, torch.float16)
    t = torch.full((9,), -100, device="cuda")
    for reduction in ("none", "sum", "mean"):
        loss, dh, dw = run(h, w, t, reduction)
        assert torch.isnan(loss).all() if reduction == "mean" else not loss.any()
        assert not dh.any() and not dw.any()
    for reduction, value in (("sum", 0.0), ("mean", float("nan"))):
        loss, dh, dw = run(h[:0], w, t[:0], reduction)
        assert loss.shape == () and (torch.isnan(loss) if value != value else loss == value) and dh.shape == (0, 64) and not dw.any()
    assert run(h[:0], w, t[:0], "none")[0].shape == (0,)


def test_targets_outside_the_vocabulary_and_nan_rows():
    h, w, t = make(150, 64, 100, torch.bfloat16, seed=6, ignored=0.0)
    clean = run(h, w, t, "none")
    t[5], t[140] = 100, -1
    h[77, 3] = float("nan")
    loss, dh, _ = run(h, w, t, "none")
    bad = torch.zeros(150, dtype=torch.bool, device="cuda")
    bad[[5, 77, 140]] = True
    assert torch.isnan(loss[bad]).all() and torch.isnan(dh[bad]).all()
    assert torch.equal(loss[~bad], clean[0][~bad]) and torch.equal(dh[~bad], clean[1][~bad])


def test_large_logits():
    """Logits of thousands: nothing overflows, a certain target has no loss."""
    w = torch.eye(64, device="cuda").half().repeat(3, 1)[:130] * 100
    t = torch.tensor([1, 2, 129], device="cuda")
    h = torch.zeros((3, 64), device="cuda").half()
    h[0, 1], h[1, 3], h[2, 1] = 100, 100, -100
    check(run(h, w, t, "none", 1.0), reference(h, w, t, "none", 1.0))


def test_strides_leading_dimensions_and_one_gradient_alone():
    from nanoquant_b200 import ops

    h, w, t = make(60, 128, 300, torch.bfloat16, seed=7)
    want = run(h, w, t)
    wide_h, wide_w = torch.randn((60, 200), device="cuda").bfloat16(), torch.randn((300, 192), device="cuda").bfloat16()
    for off in (8, 3):       # rows apart; rows that no bulk copy takes, which are copied first
        wide_h[:, off:off + 128], wide_w[:, off:off + 128] = h, w
        got = run(wide_h[:, off:off + 128], wide_w[:, off:off + 128], t)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = run(h.t().contiguous().t(), w.t().contiguous().t(), t)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    h3 = h.view(3, 20, 128).detach().requires_grad_()
    loss = ops.linear_cross_entropy(h3, w, t.view(3, 20), reduction="none")
    assert loss.shape == (3, 20) and torch.equal(loss.detach().view(-1), run(h, w, t, "none")[0])
    (dh,) = torch.autograd.grad(ops.linear_cross_entropy(h3, w, t.view(3, 20)), h3)
    assert torch.equal(dh.view(60, 128), want[1])
    wl = w.detach().requires_grad_()
    (dw,) = torch.autograd.grad(ops.linear_cross_entropy(h, wl, t), wl)
    assert torch.equal(dw, want[2])
    lazily = ops.linear_cross_entropy(torch._neg_view(-h), w, t)
    assert torch.equal(lazily, want[0]) and not lazily.requires_grad
    each = torch.linspace(-1, 1, 120, device="cuda")[::2]
    a, b = run(h, w, t, "none", each), run(h, w, t, "none", each.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_same_bits_every_time_on_two_streams_and_in_a_graph():
    from nanoquant_b200 import ops

    h, w, t = make(300, 256, 5000, torch.bfloat16, seed=8)
    want = run(h, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for i in range(4):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            outs.append(run(h, w, t))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.linear_cross_entropy(h, w, t), (h, w))
        with torch.cuda.graph(graph, stream=side):
            loss = ops.linear_cross_entropy(h, w, t)
            dh, dw = torch.autograd.grad(loss, (h, w))
    torch.cuda.current_stream().wait_stream(side)
    other = t.flip(0).contiguous()
    fresh = run(h, w, other)
    t.copy_(other)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss.detach(), fresh[0]) and torch.equal(dh, fresh[1]) and torch.equal(dw, fresh[2])


def test_capture_that_the_default_stream_holds_is_refused():
    from nanoquant_b200 import ops

    h, w, t = make(10, 64, 100, torch.bfloat16)
    w.requires_grad_()
    held = ops.linear_cross_entropy(h, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with pytest.raises(RuntimeError, match="held by an autograd graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            ops.linear_cross_entropy(h, w, t)
    assert torch.isfinite(held)


def test_such_a_capture_is_refused_for_a_padded_batch_of_hidden_states():
    """[batch, length, N] reaches the product as a view of the leaf."""
    from nanoquant_b200 import ops

    h, w, t = make(12, 64, 100, torch.bfloat16)
    h, t = h.view(3, 4, 64).requires_grad_(), t.view(3, 4)
    held = ops.linear_cross_entropy(h, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with pytest.raises(RuntimeError, match="held by an autograd graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            ops.linear_cross_entropy(h, w, t)
    assert torch.isfinite(held)


def test_training_step_captured_behind_a_warm_up_that_is_still_held():
    """The usual way to capture a training step: warm-up on a side stream, whose loss lives on while the step is captured."""
    from nanoquant_b200 import ops

    h, w, t = make(50, 128, 700, torch.bfloat16, seed=14)
    gamma = torch.ones(128, device="cuda", requires_grad=True)
    w.requires_grad_()
    step = lambda: ops.linear_cross_entropy(ops.rms_norm(h, gamma), w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            gamma.grad = w.grad = None
            loss = step()
            loss.backward()
    torch.cuda.current_stream().wait_stream(side)
    want = [loss.detach().clone(), gamma.grad.clone(), w.grad.clone()]
    gamma.grad = w.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
        captured.backward()
    for p in (gamma, w):
        p.grad.zero_()
    graph.replay()
    torch.cuda.synchronize()
    # (a captured backward pass writes a fresh gradient, as an eager one with grad = None does)
    assert all(torch.equal(a, b) for a, b in zip((captured.detach(), gamma.grad, w.grad), want))


def test_offsets_beyond_31_bits():
    N, V = 8192, 300000
    h = torch.randn((3, N), device="cuda").bfloat16()
    w = torch.zeros((V, N), dtype=torch.bfloat16, device="cuda")
    w[-2:] = (torch.randn((2, N), device="cuda") * 0.02).bfloat16()
    t = torch.tensor([V - 1, 0, -100], device="cuda")
    loss, dh, dw = run(h, w, t, "none", 1.0)
    l = h.double() @ w[-2:].double().T
    lse = torch.logsumexp(torch.cat([torch.zeros((3, V - 2), dtype=torch.float64, device="cuda"), l], 1), 1)
    each = torch.stack([lse[0] - l[0, 1], lse[1], 0 * lse[2]])
    assert ((loss.double() - each).abs() <= 1e-4).all()
    d = (l - lse[:, None]).exp()
    d[0, 1] -= 1
    d[2] = 0
    want = d.T @ h.double()
    bound = 2.0 ** -8 * (2 * d.abs().T @ h.double().abs() + want.abs())
    assert ((dw[-2:].double() - want).abs() <= bound).all()
    assert dw[0].any() and dw[V // 2].any() and not dh[2].any()


def test_refusals():
    from nanoquant_b200 import ops

    h, w, t = make(4, 64, 32, torch.float16)
    ce = ops.linear_cross_entropy
    for bad in (lambda: ce(h.float(), w.float(), t), lambda: ce(h.cpu(), w, t), lambda: ce(h, w.cpu(), t), lambda: ce(h, w.bfloat16(), t), lambda: ce(h[:, :32], w, t),
                lambda: ce(h, w, t[:3]), lambda: ce(h, w, t.float()), lambda: ce(h, w, t.cpu()), lambda: ce(h[:, :60], w[:, :60], t), lambda: ce(h, w[:0], t),
                lambda: torch.func.vmap(lambda x: ce(x, w, t[0]))(h)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        ce(h, w, t, reduction="avg")
    hr = h.detach().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(ce(hr, w, t), hr, create_graph=True)
