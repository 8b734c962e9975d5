"""What the tensor cores' cut-off sums leave in the gradients of `ops.linear_cross_entropy`.

Every matrix instruction adds 16 products to a sum and cuts all 17 off, towards zero: about 1.6 2^-23 of the sum so far, if that has one sign, so 0.8 2^-23 of the
final one.  Sums are therefore taken out of the tensor cores, logits after 32 instructions, those of the gradients after 128, and added in fp32, rounded to nearest:
an error with a sign of at most 32 or 128 times 2^-23 of a sum of one sign, whatever its length."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CUT, SUMS = 32 * 2.0 ** -23, 128 * 2.0 ** -23


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


def bias(got, want):
    """Mean relative error, and 5 standard deviations of the mean of as many uniform half steps.  Against the exact values rounded as the kernel rounds its own: what a
    type does to values that lie close together (a sum over 40000 words is 64 to 2 steps of fp16, and its steps double at 64) is then the same on both sides."""
    u = torch.finfo(got.dtype).eps / 2
    return ((got.double() - want.to(got.dtype).double()) / want).mean().item(), 5 * u / (3 * want.numel()) ** 0.5


# exponentials, lse and its product with log2(e): a few 2^-24 each, of numbers up to 16
ARITHMETIC = 8 * 2.0 ** -23


@pytest.mark.parametrize("T", [65536])
def test_long_sums_over_tokens_have_no_sign(T):
    """dw of words that are nobody's target: T positive products each."""
    N, V = 256, 512
    gen = torch.Generator(device="cuda").manual_seed(1)
    h = (torch.rand((T, N), generator=gen, device="cuda") + 0.5).half()
    w = (torch.randn((V, N), generator=gen, device="cuda") / 64).half()
    t = torch.zeros(T, dtype=torch.long, device="cuda")
    _, dw = gradients(h, w, t, 8.0)
    p = torch.softmax(h.double() @ w.double().T, 1)
    want = 8 * (p.T @ h.double())[1:]
    off, noise = bias(dw[1:], want)
    assert abs(off) <= noise + SUMS + ARITHMETIC, (off, noise)


def test_long_sums_over_words_have_no_sign():
    """dh, the target's row of the weight being zero: V positive products each."""
    T, N, V = 2048, 1024, 40000
    gen = torch.Generator(device="cuda").manual_seed(2)
    h = (torch.randn((T, N), generator=gen, device="cuda") / 64).half()
    w = (torch.rand((V, N), generator=gen, device="cuda") + 0.5).half()
    w[7] = 0
    t = torch.full((T,), 7, device="cuda")
    dh, _ = gradients(h, w, t, 64.0)
    l = h.double() @ w.double().T
    want = 64 * (torch.softmax(l, 1) @ w.double())
    off, noise = bias(dh, want)
    assert abs(off) <= noise + SUMS + ARITHMETIC, (off, noise)
