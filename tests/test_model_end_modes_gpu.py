"""The calls behind the last decoder layer under what watches or records calls: forward-mode derivatives."""
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
