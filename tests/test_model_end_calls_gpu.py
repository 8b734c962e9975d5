"""Calls behind the last decoder layer next to other calls: kernels that release the next one early."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 6, 40, 600])
def test_behind_kernels_that_release_the_next_one_early(T):
    """A quantised linear starts the kernel behind it before its outputs are written.  The same buffers again and again with other values: each step has to give
    what it gives with everything complete before every call."""
    from nanoquant_b200 import ops
    from tests.util import make_layer, tiles_on_gpu

    N, R, M, V = 1024, 256, 1024, 1000
    L = make_layer(N, R, M, T, torch.bfloat16, seed=T)
    g = torch.Generator(device="cuda").manual_seed(T)
    head = (torch.randn((V, M), generator=g, device="cuda") * 0.05).bfloat16()
    gamma = torch.ones(M, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    t = torch.randint(V, (T,), generator=g, device="cuda")
    q, s = ops.quantize_int8(head)
    v, u = tiles_on_gpu(L["V"]), tiles_on_gpu(L["U"])
    xs = [torch.randn((T, N), generator=g, device="cuda").bfloat16() for _ in range(6)]

    def step(x, wait):
        out = []
        for op in (lambda h: ops.rms_norm(h), lambda h: ops.layer_norm(h, gamma), lambda h: ops.int8_linear_forward(h, q, s), lambda h: ops.quantize_int8(h)[0],
                   lambda h: ops.linear_cross_entropy(h, head, t, reduction="none"), lambda h: ops.rms_norm(h[:, 1:])):
            h = ops.linear_forward(x, L["s_pre"], v, L["s_mid"], u, L["s_post"], R)
            if wait:
                torch.cuda.synchronize()
            out.append(op(h).detach())
        return out

    want = [step(x, True) for x in xs]
    for _ in range(20):
        for x, w in zip(xs, want):
            assert all(torch.equal(a, b) for a, b in zip(step(x, False), w))
