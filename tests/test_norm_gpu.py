"""Layer norm and RMS norm (`ops.layer_norm`, `ops.rms_norm`) against the definition in 64 bits, forward and backward.

Bounds, element by element.  An output is rounded once: half a step, `finfo.eps / 2` of its value (and half the smallest number fp16 has).  Before that
come fp32 sums: a mean adds at most 32 elements in a thread and 10 times across threads, so it is off by at most 42 roundings of 2^-24 of mean|x|;
with the few roundings behind it 2^-18 of the terms' magnitudes covers all.  Sums over the rows have up to rows / CTAs + CTAs / 8 + 8 terms one
after another, at most 200 at these sizes: 2^-16 of the sum of magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
DTYPES = [torch.float16, torch.bfloat16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def reference(x, w, b, dy, eps, center):
    """Definition in 64 bits: (y, dx, dw, db) and the magnitudes of the terms of each."""
    x, dy = x.detach().double(), dy.double()
    n = x.size(-1)
    one = torch.ones(n, dtype=torch.float64, device=x.device)
    w = one if w is None else w.detach().double()
    b = 0 * one if b is None else b.detach().double()
    m = x.mean(-1, keepdim=True) if center else torch.zeros_like(x[..., :1])
    r = 1 / (((x - m) ** 2).mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - m) * r
    g = dy * w
    c1, c2 = (g * xh).mean(-1, keepdim=True), g.mean(-1, keepdim=True) if center else 0
    size = (x.abs() + x.abs().mean(-1, keepdim=True)) * r if center else x.abs() * r
    mags = (size * w.abs() + b.abs(),
            r * (g.abs() + g.abs().mean(-1, keepdim=True) + size * (g.abs() * size).mean(-1, keepdim=True)),
            (dy.abs() * size).flatten(0, -2).sum(0), dy.abs().flatten(0, -2).sum(0))
    return (xh * w + b, r * (g - c2 - xh * c1), (dy * xh).flatten(0, -2).sum(0), dy.flatten(0, -2).sum(0)), mags


def check(got, want, mags, rels=(2.0 ** -18, 2.0 ** -17, 2.0 ** -16, 2.0 ** -16)):
    for name, t, t64, mag, rel in zip(("y", "dx", "dw", "db"), got, want, mags, rels):
        if t is None:
            continue
        bound = (half_step(t.dtype) if t.dtype != torch.float32 else 2.0 ** -24) * t64.abs() + rel * mag + TINY.get(t.dtype, 0.0)
        excess = ((t.double() - t64).abs() - bound * (1 + 2.0 ** -10)).max().item()
        assert excess <= 0, (name, excess)


def make(shape, dtype, seed=0, wdtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")
    n = shape[-1]
    x = (rand(*shape) * 2 + 0.3).to(dtype)
    return x, (1 + 0.2 * rand(n)).to(wdtype or dtype), (0.3 * rand(n)).to(wdtype or dtype), rand(*shape).to(dtype)


def run(x, w, b, dy, center, eps=1e-5):
    from nanoquant_b200 import ops

    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = ops.layer_norm(x, w, b, eps=eps) if center else ops.rms_norm(x, w, eps=eps)
    grads = list(torch.autograd.grad(y, leaves, dy))
    return [y.detach()] + [grads.pop(0) if t is not None else None for t in (x, w, b)]


@pytest.mark.parametrize("center", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [
    (1, 4096), (2, 8), (1, 1), (5, 3), (7, 33), (129, 128), (600, 512), (40, 1000), (33, 1001), (300, 1024), (50, 2048), (700, 2056),
    (297, 4096), (9, 4104), (3, 8192), (310, 8200), (5, 16384), (6, 4999), (3, 16383),
    (1201, 1), (700, 7), (333, 33), (1500, 511), (601, 1001), (400, 4097), (302, 8191), (299, 9001), (310, 16383), (2000, 640), (303, 16384), (5000, 72)])
def test_norm_matches_definition(rows, cols, dtype, center):
    x, w, b, dy = make((rows, cols), dtype, seed=rows * 7 + cols)
    b = b if center else None
    want, mags = reference(x, w, b, dy, 1e-5, center)
    check(run(x, w, b, dy, center), want, mags)


@pytest.mark.parametrize("center", [True, False])
def test_norm_without_weight_or_with_an_fp32_one(center):
    for w_on, b_on, wdtype in ((False, False, None), (True, False, torch.float32), (True, True, torch.float32)):
        x, w, b, dy = make((2, 37, 640), torch.bfloat16, seed=3, wdtype=wdtype)
        w, b = w if w_on else None, b if b_on and center else None
        want, mags = reference(x, w, b, dy, 1e-5, center)
        check(run(x, w, b, dy, center), want, mags)


def test_norm_strides():
    """Rows apart, rows that start at any address, columns that are not dense, broadcast rows and gradients."""
    from nanoquant_b200 import ops

    base, w, b, dy = make((64, 1100), torch.float16, seed=5)
    for x in (base[:, :1024], base[::2, 8:1032], base[:, 3:1003], base[:, 1::2], base[:1].expand(64, 1100), base.view(8, 8, 1100)[:, ::2]):
        n = x.size(-1)
        wn, bn = w[:n].contiguous(), b[:n].contiguous()
        d = torch.randn(x.shape, device="cuda").half()
        want, mags = reference(x, wn, bn, d, 1e-5, True)
        check(run(x.detach(), wn, bn, d, True), want, mags)
    # many rows
    base = torch.randn((700, 1100), device="cuda").half()
    for x in (base[:, :1024], base[:, 3:1003], base[:, 8:520], base[:, 1:], base[::2, 5:9]):
        n = x.size(-1)
        wn, bn = w[:n].contiguous(), b[:n].contiguous()
        d = torch.randn((*x.shape[:-1], n + 3), device="cuda").half()[..., 1:n + 1]       # gradients at any address
        want, mags = reference(x, wn, bn, d, 1e-5, True)
        check(run(x.detach(), wn, bn, d, True), want, mags)
    base = base[:64]
    # the gradient of a sum is broadcast in every dimension
    x = base[:, :1024].detach().requires_grad_()
    ops.layer_norm(x, w[:1024].contiguous().detach()).float().sum().backward()
    want, mags = reference(x, w[:1024], None, torch.ones(64, 1024, device="cuda"), 1e-5, True)
    check([None, x.grad], want[:2], mags[:2])
    # lazily negated: the memory holds the other sign
    z = torch._neg_view(base)
    assert torch.equal(ops.rms_norm(z), ops.rms_norm(-base))


def test_norm_gradient_matches_differences():
    """<dx, v> against (f(x + v) - f(x - v)) / 2 for f = <y, dy>, with steps that fp16 holds exactly."""
    from nanoquant_b200 import ops

    rows, cols = 3, 512
    x, w, b, dy = make((rows, cols), torch.float16, seed=11)
    x = (x * 64).round() / 64                       # multiples of 2^-6 below 16: x +- v is exact
    v = (torch.randint(0, 2, x.shape, device="cuda") * 2 - 1).half() / 64
    f = lambda t: (ops.layer_norm(t, w, b).double() * dy.double()).sum().item()
    dx = run(x.clone(), w.clone(), b.clone(), dy, True)[1]
    slope, diff = (dx.double() * v.double()).sum().item(), (f(x + v) - f(x - v)) / 2
    # y is rounded to 2^-11 of itself: rms error of the two sums; |v| = 2^-6 of a row's sigma of 2: third-order terms 2^-18 of the sum of |dy|
    scale = (dy.double().abs().sum()).item()
    noise = 2.0 ** -11 * (dy.double() ** 2 * ops.layer_norm(x, w, b).double() ** 2).sum().sqrt().item()
    assert abs(slope - diff) <= 4 * noise + 2.0 ** -14 * scale, (slope, diff)


def test_norm_values_that_are_not_finite_stay_in_their_row():
    from nanoquant_b200 import ops

    x, w, b, _ = make((9, 1024), torch.bfloat16, seed=2)
    clean = ops.layer_norm(x, w, b)
    x[2, 5], x[4, 1000] = float("nan"), float("inf")
    y = ops.layer_norm(x, w, b)
    bad = torch.zeros(9, dtype=torch.bool, device="cuda")
    bad[[2, 4]] = True
    assert torch.isnan(y[2]).all() and torch.isnan(y[4]).any() and torch.equal(y[~bad], clean[~bad])
    assert torch.equal(ops.rms_norm(torch.zeros_like(x)), torch.zeros_like(x))      # eps keeps a row of zeros finite
    big = torch.full((2, 4096), 60000.0, dtype=torch.float16, device="cuda")        # squares beyond fp16
    assert torch.equal(ops.rms_norm(big), torch.ones_like(big))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(3, 40), (5, 1003), (400, 256), (400, 1000), (301, 5120), (333, 5001), (600, 8200)])
def test_layer_norm_of_rows_far_from_zero(rows, cols, dtype):
    """Rows c + k step, k = 0..3, which both types hold; c up to 250 steps.  All sums of x are whole steps below 2^24 and exact; a mean is rounded once per warp
    and once over the warps, 3 2^-24 of it with what the distances between the warps' add, and x less the mean is exact.  Constant rows (k = 0) have no error."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    c = torch.randint(130, 250, (rows, 1), generator=g, device="cuda")
    k = torch.randint(0, 4, (rows, cols), generator=g, device="cuda") * (torch.arange(rows, device="cuda") % 3 > 0)[:, None]
    x = ((c + k) * 4).to(dtype)
    _, w, b, dy = make((rows, cols), dtype, seed=4)
    y, dx, dw, _ = run(x, w, b, dy, True)
    m = x.detach().double().mean(-1, keepdim=True)
    (want, _, _, _), _ = reference(x, w, b, dy, 1e-5, True)
    r = 1 / (((x.detach().double() - m) ** 2).mean(-1, keepdim=True) + 1e-5).sqrt()
    wd, bd = w.detach().double().abs(), b.detach().double().abs()
    moved = (torch.arange(rows, device="cuda") % 3 > 0)[:, None]
    bound = half_step(dtype) * want.abs() + moved * (3 * 2.0 ** -24 * m * r * wd + 2.0 ** -18 * (want.abs() + 2 * bd)) + TINY[dtype]
    excess = ((y.double() - want).abs() - bound * (1 + 2.0 ** -10)).max().item()
    assert excess <= 0, excess
    flat = run(x[::3].detach().clone(), w, b, dy[::3], True)
    assert torch.equal(flat[0], b.detach().expand_as(flat[0])) and not flat[2].any()


def test_norm_no_rows():
    from nanoquant_b200 import ops

    x = torch.empty((0, 64), dtype=torch.float16, device="cuda", requires_grad=True)
    w = torch.ones(64, dtype=torch.float16, device="cuda", requires_grad=True)
    y = ops.rms_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), y.detach())
    assert y.shape == (0, 64) and dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))


def test_norm_same_bits_every_time_and_in_a_graph():
    from nanoquant_b200 import ops

    x, w, b, dy = make((777, 2048), torch.bfloat16, seed=8)
    a, c = run(x, w, b, dy, True), run(x, w, b, dy, True)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    x, w, b = (t.detach().clone().requires_grad_() for t in (x, w, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.layer_norm(x, w, b), (x, w, b), dy)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = ops.layer_norm(x, w, b)
            grads = torch.autograd.grad(y, (x, w, b), dy)
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad():
        dy.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y.detach(), a[0]) and all(torch.equal(g, -p) for g, p in zip(grads, a[1:]))


def test_norm_refuses_a_capture_whose_gradient_the_default_stream_holds():
    from nanoquant_b200 import ops

    x, w, b, dy = make((4, 64), torch.bfloat16, seed=8)
    w.requires_grad_()
    held = ops.layer_norm(x, w, b)                  # keeps w's accumulator, made on this stream
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="held by an autograd graph"):
        with torch.cuda.graph(graph, stream=side):
            ops.layer_norm(x, w, b)
    del held
    torch.cuda.synchronize()
    assert torch.isfinite(ops.layer_norm(x, w, b)).all()


def test_norm_refuses_such_a_capture_behind_other_operations():
    """The leaf whose accumulator the default stream made need not be an argument itself."""
    from nanoquant_b200 import ops

    x, w, b, dy = make((4, 64), torch.bfloat16, seed=8)
    x.requires_grad_()
    held = ops.layer_norm(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="held by an autograd graph"):
        with torch.cuda.graph(graph, stream=side):
            ops.layer_norm(x.view(2, 2, 64) * 2, w, b)
    del held
    torch.cuda.synchronize()
    assert torch.isfinite(ops.layer_norm(x, w, b)).all()


def test_norm_offsets_beyond_31_bits():
    from nanoquant_b200 import ops

    rows, cols = 140000, 16384
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    x[-2:] = torch.randn((2, cols), device="cuda").bfloat16()
    y = ops.rms_norm(x)
    assert torch.equal(y[-2:], ops.rms_norm(x[-2:].clone())) and not y[0].any()


def test_norm_refusals():
    from nanoquant_b200 import _lib, ops

    x, w, b, dy = make((4, 64), torch.float16)
    for bad in (lambda: ops.rms_norm(x.float()), lambda: ops.rms_norm(x.cpu()), lambda: ops.layer_norm(x, w.cpu()), lambda: ops.layer_norm(x, w[:32]),
                lambda: ops.layer_norm(x, w, b.float()), lambda: ops.layer_norm(x, None, b), lambda: ops.layer_norm(x, w.bfloat16()),
                lambda: ops.rms_norm(x[0, 0]), lambda: torch.func.vmap(ops.rms_norm)(x)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(_lib.NanoQuantError) as e:
        ops.rms_norm(torch.zeros((1, _lib.lib().nq_norm_max_columns() + 1), dtype=torch.float16, device="cuda"))
    assert e.value.status == _lib.NQ_ERR_TOO_LARGE
    x.requires_grad_()
    (g,) = torch.autograd.grad(ops.rms_norm(x).sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(ops.rms_norm(x).sum(), x, create_graph=True)
