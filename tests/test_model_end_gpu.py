"""What stands behind the last decoder layer, together: a decode step's end (quantised linear with its residual, norm, 8-bit head) and a step of training the
final norm and the head on frozen hidden states."""
import pytest
import torch

from tests.util import make_layer, tiles_on_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 16, 200])
def test_decode_step_end(T):
    from nanoquant_b200 import ops

    N, R, M, V = 1024, 256, 1024, 3001
    L = make_layer(N, R, M, T, torch.bfloat16, seed=T)
    g = torch.Generator(device="cuda").manual_seed(1)
    resid = torch.randn((T, M), generator=g, device="cuda").bfloat16()
    head = (torch.randn((V, M), generator=g, device="cuda") * 0.03).bfloat16()
    q, s = ops.quantize_int8(head)
    v, u = tiles_on_gpu(L["V"]), tiles_on_gpu(L["U"])

    def step():
        h = ops.linear_forward(L["x"], L["s_pre"], v, L["s_mid"], u, L["s_post"], R, residual=resid)
        n = ops.rms_norm(h)
        return h, n, ops.int8_linear_forward(n, q, s)

    h, n, y = step()
    h64 = h.double()
    n64 = h64 / (h64.square().mean(1, keepdim=True) + 1e-6).sqrt()
    assert ((n.double() - n64).abs() <= 2.0 ** -8 * n64.abs() + 2.0 ** -17).all()
    top = n.double().abs().amax(1, keepdim=True)
    y64 = ((n.double() * 127 / top).round() @ q.double().T) * (top / 127) * s.double()
    assert ((y.double() - y64).abs() <= (2.0 ** -8 + 2.0 ** -20) * y64.abs()).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _, _, out = step()
    L["x"].neg_()
    want = step()[2]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_training_step_of_norm_and_head():
    """Gradients of the norm's weight and bias through the loss, against the whole step in 64 bits."""
    from nanoquant_b200 import ops

    T, N, V = 333, 512, 2000
    g = torch.Generator(device="cuda").manual_seed(2)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")
    x, w, b, head = rand(T, N).bfloat16(), (1 + 0.1 * rand(N)), 0.1 * rand(N), (rand(V, N) * 0.05).bfloat16()
    t = torch.randint(V, (T,), generator=g, device="cuda")
    t[::5] = -100
    leaves = [v.requires_grad_() for v in (w, b, head)]
    loss = ops.linear_cross_entropy(ops.layer_norm(x, w, b), head, t)
    loss.backward()
    d = [v.detach().double().requires_grad_() for v in leaves]
    ref = torch.nn.functional.cross_entropy(torch.nn.functional.layer_norm(x.double(), (N,), d[0], d[1], 1e-5) @ d[2].T, t)
    ref.backward()
    # hidden states and their gradient are rounded to bf16 on the way, d is too: three independent half steps of 2^-8, and a loss of its first-order part
    assert abs(loss.item() - ref.item()) <= 2.0 ** -8 * abs(ref.item())
    for v, r in zip(leaves, d):
        assert v.grad.dtype == v.dtype
        assert (v.grad.double() - r.grad).norm() <= 4 * 2.0 ** -8 * r.grad.norm()
