"""The calls behind the last decoder layer under what watches or records calls: forward-mode derivatives, ``torch.jit.trace`` and ``torch.compile``."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(T, N, V, seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")
    t = torch.randint(V, (T,), generator=g, device="cuda")
    t[::4] = -100
    return rand(T, N).to(dtype), (rand(V, N) * 0.05).to(dtype), t, (1 + 0.1 * rand(N)).to(dtype), (0.1 * rand(N)).to(dtype)


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    """No call has a forward derivative; an output without a tangent would say that it is zero."""
    import torch.autograd.forward_ad as fwad
    from nanoquant_b200 import ops

    h, head, t, w, b = make(6, 64, 40)
    if grad:
        for v in (h, head, w, b):
            v.requires_grad_()
    calls = [(h, lambda d: ops.rms_norm(d, w)), (w, lambda d: ops.rms_norm(h, d)), (h, lambda d: ops.layer_norm(d, w, b)), (b, lambda d: ops.layer_norm(h, w, d)),
             (h, lambda d: ops.rms_norm(d.t())[:0]), (h, lambda d: ops.linear_cross_entropy(d, head, t)), (head, lambda d: ops.linear_cross_entropy(h, d, t)),
             (h, lambda d: ops.linear_cross_entropy(d.view(2, 3, 64), head, t.view(2, 3)))]
    for v, call in calls:
        with fwad.dual_level():
            with pytest.raises(RuntimeError, match="forward"):
                call(fwad.make_dual(v, torch.ones_like(v)))
        call(v)                                     # (and without a tangent as ever)


def traced_calls(ops, head, t, w, b):
    q, s = ops.quantize_int8(head)
    bias = torch.linspace(-1, 1, head.size(0), device="cuda").to(head.dtype)
    return {
        "rms": lambda x: ops.rms_norm(x, w), "rms_plain": lambda x: ops.rms_norm(x), "layer": lambda x: ops.layer_norm(x, w, b),
        "quantize": lambda x: ops.quantize_int8(x), "int8": lambda x: ops.int8_linear_forward(x, q, s, bias), "dense": lambda x: ops.dense_gemv_forward(x, head, bias),
        "loss": lambda x: ops.linear_cross_entropy(x, head, t), "each": lambda x: ops.linear_cross_entropy(x, head, t, reduction="none"),
        "chain": lambda x: ops.int8_linear_forward(ops.rms_norm(x * 2, w), q, s) + 1,
    }


@pytest.mark.parametrize("name", ["rms", "rms_plain", "layer", "quantize", "int8", "dense", "loss", "each", "chain"])
def test_trace_records_the_call(name):
    """What is traced has to follow its input; an output baked in as a constant would be the example's for ever."""
    from nanoquant_b200 import ops

    x, head, t, w, b = make(8, 64, 40, seed=1)
    fn = traced_calls(ops, head, t, w, b)[name]
    with torch.no_grad():
        traced = torch.jit.trace(fn, (x,))
        for y in (x, x.flip(0).contiguous() * 1.5):
            got, want = traced(y), fn(y)
            for p, r in zip(got, want) if isinstance(want, tuple) else ((got, want),):
                assert torch.equal(p, r) and p.shape == r.shape


def test_trace_records_a_quantised_linear():
    """The module's own short way is not taken while it is traced."""
    from tests.test_model_gpu import oc, fill
    from nanoquant_b200.modules.linear import NanoQuantLinear

    lin = NanoQuantLinear(256, 128, 64, has_scale_mid=True)
    fill(lin, oc.synth_linear(256, 64, 128, 2, seed=3))
    lin = lin.cuda()
    lin._prepare_kernel("gemv", torch.bfloat16)
    x = torch.randn(2, 256, device="cuda").bfloat16()
    with torch.no_grad():
        traced = torch.jit.trace(lambda x: lin(x), (x,))
        for y in (x, x * 1.5):
            assert torch.equal(traced(y), lin(y))


def test_trace_of_what_is_no_operator_is_refused():
    """Launch groups, and linears with a bias or residual: a trace would hold constants, or memory that nobody fills."""
    from tests.test_model_gpu import oc, fill
    from nanoquant_b200 import ops
    from nanoquant_b200.modules.group import LinearGroup
    from nanoquant_b200.modules.linear import NanoQuantLinear

    lins = []
    for bias in (False, False, True):
        lin = NanoQuantLinear(256, 128, 64, has_scale_mid=True)
        fill(lin, oc.synth_linear(256, 64, 128, 2, seed=3))
        lin = lin.cuda()
        if bias:
            lin.bias = torch.nn.Parameter(torch.randn(128, device="cuda").bfloat16(), requires_grad=False)
        lin._prepare_kernel("gemv", torch.bfloat16)
        lins.append(lin)
    group = LinearGroup(lins[:2])
    s_in, v, s_mid, u, s_out, rank, _ = lins[0].launch_operands()
    x = torch.randn(2, 256, device="cuda").bfloat16()
    with torch.no_grad():
        for fn in (lambda x: lins[2](x), lambda x: group(x)[1], lambda x: ops.linear_forward(x, s_in, v, s_mid, u, s_out, rank),
                   lambda x: ops.gemv_forward(x, s_in, v, s_mid, u, s_out, rank)):
            assert torch.isfinite(fn(x)).all()
            with pytest.raises(RuntimeError, match="cannot be traced"):
                torch.jit.trace(fn, (x,))
            assert torch.isfinite(fn(x)).all()


@pytest.mark.parametrize("name", ["rms", "rms_plain", "layer", "quantize", "int8", "dense", "loss", "each", "chain"])
def test_one_graph_under_torch_compile(name):
    from nanoquant_b200 import ops

    x, head, t, w, b = make(8, 64, 40, seed=2)
    ops.reserve_scratch(x.device, 256)
    fn = traced_calls(ops, head, t, w, b)[name]
    torch._dynamo.reset()
    with torch.no_grad():
        for kw in (dict(backend="aot_eager"), dict(mode="reduce-overhead")):
            compiled = torch.compile(fn, fullgraph=True, **kw)
            for y in (x, x.flip(0).contiguous() * 1.5, x, x * 0.5):
                want, got = fn(y), compiled(y)
                for p, r in zip(got, want) if isinstance(want, tuple) else ((got, want),):
                    assert torch.equal(p, r) and p.stride() == r.stride()


def test_rows_apart_under_torch_compile():
    """Inputs that are no dense tensors, three dimensions, and a weight in 8 bits whose rows are padded."""
    from nanoquant_b200 import ops

    base, head, t, w, b = make(24, 520, 40, seed=3)
    base = base.view(4, 6, 520)
    q, s = ops.quantize_int8(head[:, 3:503])
    t = t.view(4, 6)
    assert q.stride(0) == 512
    ops.reserve_scratch(base.device, 256)

    def fn(x):
        h = x[..., 3:503]
        n = ops.layer_norm(h, w[3:503].contiguous(), b[3:503].contiguous())
        return n, ops.int8_linear_forward(n, q, s), ops.linear_cross_entropy(x, head, t, reduction="none")

    torch._dynamo.reset()
    with torch.no_grad():
        got, want = torch.compile(fn, fullgraph=True, backend="aot_eager")(base), fn(base)
    assert all(torch.equal(p, r) and p.shape == r.shape for p, r in zip(got, want))


@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("bias", [False, True])
def test_training_step_under_torch_compile(reduction, bias):
    """Gradients of the compiled step: the same kernels, so the same bits."""
    from nanoquant_b200 import ops

    x, head, t, w, b = make(40, 128, 300, seed=4)

    def step(x, w, b, head):
        h = ops.layer_norm(x, w, b) if bias else ops.rms_norm(x, w.float())
        return ops.linear_cross_entropy(h, head, t, reduction=reduction).sum()

    leaves = [v.requires_grad_() for v in ((x, w, b, head) if bias else (x, w, head))]
    torch._dynamo.reset()
    want = torch.autograd.grad(step(x, w, b, head), leaves)
    loss = torch.compile(step, fullgraph=True, backend="aot_eager")(x, w, b, head)
    got = torch.autograd.grad(loss, leaves)
    assert torch.equal(loss, step(x, w, b, head)) and all(torch.equal(p, r) for p, r in zip(got, want))
    loss = torch.compile(step, fullgraph=True, backend="aot_eager")(x, w, b, head.detach())      # one leaf without a gradient
    got = torch.autograd.grad(loss, leaves[:-1])
    assert all(torch.equal(p, r) for p, r in zip(got, want))


def test_refusals_under_torch_compile():
    from nanoquant_b200 import ops

    x, head, t, w, b = make(8, 64, 40)
    q, s = ops.quantize_int8(head)
    for bad in (lambda x: ops.rms_norm(x.float()), lambda x: ops.layer_norm(x, w[:32]), lambda x: ops.layer_norm(x, w, b.float()), lambda x: ops.int8_linear_forward(x, q, s[:-1]),
                lambda x: ops.linear_cross_entropy(x, head, t[:3]), lambda x: ops.linear_cross_entropy(x[:, :60], head[:, :60], t)):
        torch._dynamo.reset()
        with pytest.raises(Exception):
            torch.compile(bad, fullgraph=True, backend="aot_eager")(x)
    with pytest.raises(RuntimeError, match="differentiable once"):       # as in an eager call
        y = torch.ops.nanoquant_b200.norm(x.requires_grad_(), w, None, 1e-6, False)[0]
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_registrations_of_the_operators():
    """Schemas, shapes for tracing (also with sizes that are not known) and derivatives are those of what runs."""
    x, head, t, w, b = make(8, 64, 40, seed=5)
    op = torch.ops.nanoquant_b200
    grad = lambda *ts: tuple(v.detach().clone().requires_grad_() for v in ts)
    from nanoquant_b200 import ops

    q, s = ops.quantize_int8(head)
    y, stats = op.norm(x, w, b, 1e-5, True)
    loss, lse, count = op.linear_cross_entropy(x, head, t, -100, 2)
    for f, args in ((op.norm, (x, None, None, 1e-6, False)), (op.norm, (*grad(x, w, b), 1e-5, True)), (op.norm_backward, (y, x, w, stats, True, [True, True, True])),
                    (op.norm_backward, (y, x, w, stats, True, [False, True, False])), (op.quantize_rows, (x.view(2, 4, 64)[..., :50],)), (op.int8_linear, (x.view(2, 4, 64), q, s, None)),
                    (op.dense_gemv, (x, head, None)), (op.linear_cross_entropy, (x, head, t, -100, 2)), (op.linear_cross_entropy, (*grad(x, head), t, -100, 1)),
                    (op.linear_cross_entropy_backward, (torch.ones_like(loss), x, head, t, lse, count, -100, 2, [True, False]))):
        torch.library.opcheck(f.default, args, test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_dynamic"))
