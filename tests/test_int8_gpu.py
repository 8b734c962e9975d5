"""The head in 8 bits (`ops.quantize_int8`, `ops.int8_linear_forward`) against its definition in 64 bits.

The quantised values are exact: 127 x / max|x| of 16-bit x is a half exactly (63.5 for x = max|x| / 2), or at least 2^-12 away from one, which the rounding
of an fp32 quotient below 128 cannot cross.  The sums are exact whole numbers; their conversion, the scales' product, its application and the bias are four roundings of 2^-24 (2^-21
covers them), the scale's own one is part of the definition (fp32), and the output is rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
DTYPES = [torch.float16, torch.bfloat16]


def quantized(x):
    """(q, scale) of the definition: q in 64 bits, the scale as fp32."""
    top = x.double().abs().amax(-1)
    return (x.double() * 127 / torch.where(top > 0, top, 1.0)[..., None]).round(), (top.float() / torch.tensor(127.0, device=x.device)).double()


def expected(x, q, s, b):
    xq, xs = quantized(x)
    y = xq @ q.double().T
    return y * xs[:, None] * s.double() + (0 if b is None else b.double())


def check(y, y64, b):
    mag = y64.abs() + (0 if b is None else b.double().abs())
    bound = torch.finfo(y.dtype).eps / 2 * y64.abs() + 2.0 ** -21 * mag + TINY[y.dtype]
    excess = ((y.double() - y64).abs() - bound * (1 + 2.0 ** -10)).max().item()
    assert excess <= 0, excess


def make(T, N, V, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")
    return rand(T, N).to(dtype), (rand(V, N) * 0.02).to(dtype), (rand(V) * 0.5).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 17), (5, 1003), (64, 4096), (2, 40000), (400, 128), (301, 1024), (300, 4104), (3, 16384), (2, 16392), (2, 32768)])
def test_quantize_is_exact(rows, cols, dtype):
    from nanoquant_b200 import ops

    x, _, _ = make(rows, cols, 1, dtype, seed=cols)
    x[0, 0] = 0 if cols > 1 else 3
    x[-1, :] *= 0 if rows > 1 else 1
    q, s = ops.quantize_int8(x)
    q64, s64 = quantized(x)
    assert torch.equal(q.double(), q64) and torch.equal(s.double(), s64)
    assert q.stride(0) % 16 == 0 and q.shape == x.shape and s.shape == (rows,)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_all_quotients(dtype):
    """Every ratio of two significands, at ordinary magnitudes, the smallest and the largest: halves and their neighbours among them."""
    from nanoquant_b200 import ops

    bits = 8 if dtype == torch.bfloat16 else 11
    x = torch.arange(1, 2 ** bits, device="cuda").double()
    tops = (2 ** bits - 1 - torch.arange(0, 2 ** (bits - 1), 1 if bits == 8 else 13, device="cuda")).double()
    for scale in (1.0, 2.0 ** -133, 2.0 ** 100) if dtype == torch.bfloat16 else (1.0, 2.0 ** -24, 2.0 ** 4):
        m = torch.minimum(x, tops[:, None]) * scale        # every row: all values up to its largest
        m[:, ::2] *= -1
        m = m.to(dtype)
        q, s = ops.quantize_int8(m)
        q64, s64 = quantized(m)
        assert torch.equal(q.double(), q64) and torch.equal(s.double(), s64)


def test_quantize_ties_go_to_even():
    from nanoquant_b200 import ops

    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -126.5]], device="cuda").half()
    q, s = ops.quantize_int8(x)
    assert s.item() == 1.0 and q[0].tolist() == [127, 0, 2, 2, 0, -2, 126, -126]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,V,bias", [
    (1, 1, 1, True), (2, 260, 77, True), (4, 1001, 40, False), (5, 384, 300, False), (9, 640, 200, True), (15, 4100, 64, False), (16, 6144, 50, True),
    (16, 6272, 50, False), (8, 12288, 70, False), (8, 12300, 33, False), (1, 4096, 512, False), (1, 16, 4, False), (3, 100, 33, False), (8, 128, 16, False), (37, 1003, 777, True), (127, 64, 130, True), (128, 256, 300, False),
    (129, 512, 1000, True), (255, 200, 31, False), (257, 2048, 513, False), (16, 2048, 40001, False), (300, 1024, 2050, True),
    (1030, 4096, 1536, False), (2, 16384, 100, False)])
def test_linear_matches_definition(T, N, V, bias, dtype):
    from nanoquant_b200 import ops

    x, w, b = make(T, N, V, dtype, seed=T + N)
    b = b if bias else None
    q, s = ops.quantize_int8(w)
    y = ops.int8_linear_forward(x, q, s, b)
    assert y.shape == (T, V) and y.dtype == dtype
    check(y, expected(x, q, s, b), b)



def test_linear_extreme_sums_are_exact():
    """Every product 127 * 127: the longest sum fits 32 bits and is exact to its last unit."""
    from nanoquant_b200 import ops

    N = 131072
    x = torch.ones((2, N), dtype=torch.bfloat16, device="cuda")
    x[1, ::2] = -1
    q = torch.full((16, N), 127, dtype=torch.int8, device="cuda")
    q[1:, 0] = torch.arange(15, device="cuda").to(torch.int8)
    y = ops.int8_linear_forward(x, q, torch.ones(16, device="cuda"))
    check(y, expected(x, q, torch.ones(16, device="cuda"), None), None)
    with pytest.raises(Exception) as e:
        ops.int8_linear_forward(torch.ones((1, N + 16), dtype=torch.bfloat16, device="cuda"),
                                torch.zeros((1, N + 16), dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))
    assert e.value.status == -9


def test_linear_shapes_strides_and_streams():
    from nanoquant_b200 import ops

    x, w, b = make(24, 520, 300, torch.bfloat16, seed=4)
    q, s = ops.quantize_int8(w)
    want = ops.int8_linear_forward(x, q, s, b)
    assert torch.equal(ops.int8_linear_forward(x.view(2, 3, 4, 520), q, s, b).view(24, 300), want)
    wide = torch.randn((24, 700), device="cuda").bfloat16()
    wide[:, 3:523] = x
    assert torch.equal(ops.int8_linear_forward(wide[:, 3:523], q, s, b), want)              # rows apart, at any address
    assert torch.equal(ops.int8_linear_forward(x.t().contiguous().t(), q, s, b), want)      # columns that are not dense
    assert torch.equal(ops.int8_linear_forward(torch._neg_view(-x), q, s, b), want)
    assert torch.equal(ops.int8_linear_forward(x[0], q, s, b), want[0])
    some = torch.empty(301, device="cuda")
    some[1:] = s
    assert torch.equal(ops.int8_linear_forward(x, q, some[1:], b), want)                    # scales at any address
    assert ops.int8_linear_forward(x[:0], q, s, b).shape == (0, 300)
    one, _ = ops.quantize_int8(w[:1])
    assert torch.equal(ops.int8_linear_forward(x, one, s[:1]), ops.int8_linear_forward(x, q, s)[:, :1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for i in range(8):                                   # two streams at once, each with its own buffers
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            outs.append(ops.int8_linear_forward(x, q, s, b))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_linear_any_token_alone():
    """A token's outputs do not depend on the others, nor on how many there are."""
    from nanoquant_b200 import ops

    x, w, _ = make(300, 1024, 500, torch.float16, seed=9)
    q, s = ops.quantize_int8(w)
    y = ops.int8_linear_forward(x, q, s)
    for n in (1, 2, 100, 129):
        assert torch.equal(ops.int8_linear_forward(x[:n], q, s), y[:n])


def test_linear_values_that_are_not_finite_stay_in_their_token():
    from nanoquant_b200 import ops

    x, w, b = make(6, 256, 100, torch.bfloat16, seed=1)
    q, s = ops.quantize_int8(w)
    clean = ops.int8_linear_forward(x, q, s, b)
    x[1, 7], x[3, 0], x[4, 255] = float("nan"), float("inf"), -float("inf")
    y = ops.int8_linear_forward(x, q, s, b)
    bad = torch.tensor([False, True, False, True, True, False], device="cuda")
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])
    assert torch.equal(ops.int8_linear_forward(torch.zeros_like(x), q, s, b), b.expand(6, 100))


def test_linear_offsets_beyond_31_bits():
    from nanoquant_b200 import ops

    N, V = 16384, 140000
    q = torch.zeros((V, N), dtype=torch.int8, device="cuda")
    q[-3:] = torch.randint(-127, 128, (3, N), device="cuda").to(torch.int8)
    s = torch.ones(V, device="cuda")
    x, _, _ = make(2, N, 1, torch.bfloat16)
    y = ops.int8_linear_forward(x, q, s)
    check(y[:, -3:], expected(x, q[-3:], s[-3:], None), None)
    assert not y[:, :-3].any()
    T, V = 20000, 110000                                  # outputs beyond 2^31
    x = torch.zeros((T, 16), dtype=torch.bfloat16, device="cuda")
    x[-1, 0] = 1
    y = ops.int8_linear_forward(x, q[:1, :16].expand(V, 16).contiguous() * 0 + 1, torch.ones(V, device="cuda"))
    assert (y[-1] == 1).all() and not y[-2].any()


def test_linear_in_two_cuda_graphs_at_once():
    from nanoquant_b200 import ops

    x, w, b = make(40, 512, 1000, torch.bfloat16, seed=6)
    q, s = ops.quantize_int8(w)
    want = [ops.int8_linear_forward(v, q, s, b) for v in (x, -x)]
    ops.int8_linear_forward(x[:1], q, s, b)
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for v, st in zip((x, -x), streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(ops.int8_linear_forward(v, q, s, b))
        graphs.append(g)
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, v) for o, v in zip(outs, want))


def test_wait_that_runs_out():
    """The epilogue of a tile waits for its main loop, 250 us; with a limit of one attempt after the first (10 us in all) it gives up.  The launch ends all the
    same, drains what is in flight, gives its tensor memory back and reports; the next one on a zeroed status word is right."""
    from nanoquant_b200 import _lib, ops

    L = _lib.lib()
    T, N, V = 256, 131072, 256
    x, w, _ = make(T, N, V, torch.bfloat16, seed=2)
    q, s = ops.quantize_int8(w)
    y = torch.empty((T, V), dtype=torch.bfloat16, device="cuda")
    nb = L.nq_int8_linear_scratch_bytes(T, N)
    scratch, header = torch.empty(nb, dtype=torch.uint8, device="cuda"), torch.zeros(256, dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    call = lambda: _lib.check(L.nq_int8_linear_fwd(x.data_ptr(), q.data_ptr(), s.data_ptr(), None, y.data_ptr(), scratch.data_ptr(), nb, header.data_ptr(),
                                                   T, N, V, N, q.stride(0), V, _lib.NQ_BF16, st), "nq_int8_linear_fwd")
    status = lambda: L.nq_scratch_status(header.data_ptr(), st)
    call()
    assert status() == 0
    check(y, expected(x, q, s, None), None)
    old = L.nq_gemm_set_wait_limit(1)
    try:
        call()
        assert status() == _lib.NQ_ERR_TIMEOUT
    finally:
        assert L.nq_gemm_set_wait_limit(old) == 1
    header.zero_()
    call()
    assert status() == 0
    check(y, expected(x, q, s, None), None)


def test_linear_against_the_dense_head():
    """Near the 16-bit head it stands in for: each factor is off by at most half a step of max / 127."""
    from nanoquant_b200 import ops

    x, w, _ = make(4, 2048, 4000, torch.bfloat16, seed=12)
    y8, y16 = ops.int8_linear_forward(x, *ops.quantize_int8(w)).double(), ops.dense_gemv_forward(x, w).double()
    sx, sw = x.double().abs().amax(1, keepdim=True) / 254, w.double().abs().amax(1) / 254
    bound = sx * w.double().abs().sum(1) + x.double().abs().sum(1, keepdim=True) * sw + 2048 * sx * sw
    assert ((y8 - y16).abs() <= bound + 2.0 ** -8 * (y8.abs() + y16.abs())).all()


def test_refusals():
    from nanoquant_b200 import ops

    x, w, b = make(2, 64, 32, torch.float16)
    q, s = ops.quantize_int8(w)
    for bad in (lambda: ops.int8_linear_forward(x.float(), q, s), lambda: ops.int8_linear_forward(x.cpu(), q, s), lambda: ops.int8_linear_forward(x, q.cpu(), s),
                lambda: ops.int8_linear_forward(x[:, :32], q, s), lambda: ops.int8_linear_forward(x, q, s[:-1]), lambda: ops.int8_linear_forward(x, q, s.half()),
                lambda: ops.int8_linear_forward(x, q, s, b.bfloat16()), lambda: ops.int8_linear_forward(x, q, s, b[:5]), lambda: ops.int8_linear_forward(x, w, s),
                lambda: ops.int8_linear_forward(x[:, :60], q[:, 4:], s), lambda: ops.int8_linear_forward(x[:, :40], q.reshape(-1)[:1600].view(40, 40), s[:40]),
                lambda: ops.int8_linear_forward(x, q[:0], s[:0]), lambda: ops.quantize_int8(x.float()), lambda: ops.quantize_int8(x.cpu()),
                lambda: ops.quantize_int8(x[:, :0])):
        with pytest.raises(RuntimeError):
            bad()
