"""8-bit rows and products over the whole range of bf16: magnitudes whose products with 127 fp32 does not hold, and scales whose product it does not hold."""
import pytest
import torch

from tests.test_int8_gpu import expected, quantized

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [255, 256, 264, 1024])
def test_quantize_all_quotients_at_the_largest_magnitudes(cols):
    """Every ratio of two significands with rows whose largest value is up to the largest of bf16: 255 2^120.  Wide enough for single values, for packs of
    eight, and for packs with zeros (255 columns: rows that no 16-byte load takes)."""
    from nanoquant_b200 import ops

    tops = torch.arange(255, 127, -1, device="cuda").double()
    x = torch.zeros(cols, dtype=torch.float64, device="cuda")
    x[:255] = torch.arange(1, 256, device="cuda")
    for scale in (2.0 ** 120, 2.0 ** 119, 2.0 ** 113, 2.0 ** 112):
        m = torch.minimum(x, tops[:, None]) * scale
        m[:, ::2] *= -1
        m = m.bfloat16()
        assert torch.isfinite(m).all()
        q, s = ops.quantize_int8(m)
        q64, s64 = quantized(m)
        assert torch.equal(q.double(), q64) and torch.equal(s.double(), s64)


@pytest.mark.parametrize("T", [1, 2, 5, 200])
@pytest.mark.parametrize("N", [96, 99])
def test_linear_of_the_largest_tokens(T, N):
    """One and two tokens are quantised by the product itself, more before it; 16-byte loads and single values."""
    from nanoquant_b200 import ops

    x = torch.zeros((T, N), dtype=torch.bfloat16, device="cuda")
    x[:, 0], x[:, 1], x[:, 9], x[:, 20] = 3e38, 1.5e38, -2.9e38, 1e35
    w = torch.randint(-127, 128, (40, N), device="cuda").to(torch.int8)
    q = torch.zeros((40, 112), dtype=torch.int8, device="cuda")
    q[:, :N] = w
    s = torch.full((40,), 2.0 ** -40, device="cuda")
    y, want = ops.int8_linear_forward(x, q[:, :N], s), expected(x, w, s, None)
    # exact sums; a few roundings of 2^-24, and the output's own of half a step: bf16 has 8 significant bits, so 2^-8 of a value just above a power of two
    assert ((y.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -21) * want.abs()).all()


@pytest.mark.parametrize("T", [1, 3, 200])
def test_linear_where_the_product_of_the_scales_leaves_fp32(T):
    """s_x s_w overflows, or falls below the normal numbers, where the result does not: the sum is multiplied by one scale and then by the other."""
    from nanoquant_b200 import ops

    N, V = 64, 24
    q = torch.zeros((V, N), dtype=torch.int8, device="cuda")
    q[1::2, :32] = 127
    b = torch.randn(V, device="cuda").bfloat16()
    x = torch.full((T, N), 2.0 ** 120, dtype=torch.bfloat16, device="cuda")
    x[:, 16:32] = -x[:, :16]                       # sums of zero
    s = torch.full((V,), 2.0 ** 20, device="cuda")
    assert torch.equal(ops.int8_linear_forward(x, q, s, b), b.expand(T, V))
    x = torch.full((T, N), 2.0 ** -105, dtype=torch.bfloat16, device="cuda")
    s = torch.full((V,), 2.0 ** -32, device="cuda")
    y, want = ops.int8_linear_forward(x, q, s), expected(x, q, s, None)
    assert want.max() > 2.0 ** -126 and ((y.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -21) * want).all()
