"""What the tensor cores' cut-off sums leave in the gradients of `ops.linear_cross_entropy`.

Every matrix instruction adds 16 products to a sum and cuts all 17 off, towards zero: about 1.6 2^-23 of the sum so far, if that has one sign, so 0.8 2^-23 of the
final one.  Sums are therefore taken out of the tensor cores, logits after 32 instructions, and added in fp32, rounded to nearest: an
error with a sign of at most 32 times 2^-23 of a sum of one sign, whatever its length."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CUT = 32 * 2.0 ** -23


def gradients(h, w, t, g):
    from nanoquant_b200 import ops

    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = ops.linear_cross_entropy(h, w, t, reduction="sum")
    return torch.autograd.grad(loss, (h, w), torch.tensor(g, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 40, 300])
@pytest.mark.parametrize("N", [512, 4096, 8192])
def test_gradient_of_near_certain_targets(T, N, dtype):
    """The target's logit is 8, the others are 0: d[target] = p - 1 is about -1e-3, and has to have that size's precision.  Its logits have to be those that
    lse came from, to the bit: p is then off by the fp32 arithmetic alone, six roundings of numbers up to 16 (2^-21 each) and an exponential of 2^-21."""
    gen = torch.Generator(device="cuda").manual_seed(N + T)
    rand = lambda *s: torch.rand(s, generator=gen, device="cuda") + 0.5
    h = rand(T, N).to(dtype)
    w = torch.zeros((4, N), dtype=dtype, device="cuda")
    w[1] = (rand(N) * (8 / N)).to(dtype)
    t = torch.ones(T, dtype=torch.long, device="cuda")
    dh, _ = gradients(h, w, t, 64.0)
    l = h.double() @ w.double().T
    d = -64 * (1 - torch.softmax(l, 1)[:, 1])
    got, want = dh.double() @ w[1].double() / (w[1].double() ** 2).sum(), d
    # d and dh are rounded to the type; the logits' own error moves 1 - p by its size, relative to it
    u = torch.finfo(dtype).eps / 2
    bound = 64 * 7 * 2.0 ** -21 + want.abs() * (2 * u + 2 * (CUT + 2.0 ** -22) * 9) + (2.0 ** -25 / w[1].double().abs().min() if dtype == torch.float16 else 0)
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / want.abs()).max()
