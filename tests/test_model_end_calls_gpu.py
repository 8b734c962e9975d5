"""Calls behind the last decoder layer next to other calls: host threads, scratch of their own, kernels that release the next one early."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols,other", [((4001, 4001), (1100, 1300)), ((4096, 2056), (256, 520))])
def test_norms_of_different_widths_in_two_threads(cols, other):
    """Both threads use the same kernels with other sizes of shared memory."""
    from nanoquant_b200 import _lib

    L = _lib.lib()
    rows = 400
    errors, gate = [], threading.Barrier(2)

    def work(widths, seed):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            sets = []
            for n in widths:
                x = torch.randn((rows, n), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").bfloat16()
                sets.append((n, x, torch.empty_like(x), torch.empty((rows, 2), device="cuda"), torch.empty_like(x)))
        torch.cuda.synchronize()
        gate.wait()
        for i in range(4000):
            n, x, y, stats, dx = sets[i % 2]
            st = L.nq_norm_fwd(x.data_ptr(), None, None, y.data_ptr(), stats.data_ptr(), rows, n, n, n, 1e-5, 1, _lib.NQ_BF16, _lib.NQ_BF16, stream.cuda_stream)
            st2 = L.nq_norm_bwd(y.data_ptr(), x.data_ptr(), None, stats.data_ptr(), dx.data_ptr(), None, None, None, 0, rows, n, n, n, n, 1, _lib.NQ_BF16, _lib.NQ_BF16,
                                stream.cuda_stream)
            if st or st2:
                errors.append((n, st, st2, L.nq_last_cuda_error()))
                return
        stream.synchronize()
        for n, x, y, _, _ in sets:
            d = x.double()
            want = (d - d.mean(1, keepdim=True)) / (d.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
            if not ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -17).all():
                errors.append((n, "values"))

    threads = [threading.Thread(target=work, args=a) for a in ((cols, 1), (other, 2))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors[:2]


def test_backward_keeps_the_scratch_of_its_forward():
    """The backward pass runs on a thread of autograd's; its status word is the one that the forward call was given, also when the caller has left the block."""
    from nanoquant_b200 import _lib, ops

    dev = torch.cuda.current_device()
    h = torch.randn((20, 64), device="cuda").bfloat16().requires_grad_()
    w = torch.randn((100, 64), device="cuda").bfloat16()
    t = torch.arange(20, device="cuda")
    want = torch.autograd.grad(ops.linear_cross_entropy(h, w, t), h)[0]
    shared = ops._scratch.pop(dev)
    _lib.ext().set_scratch(dev, 0, 0)
    try:
        mine = torch.zeros(4096, dtype=torch.uint8, device="cuda")
        with ops.private_scratch(mine):
            loss = ops.linear_cross_entropy(h, w, t)
        address = mine.data_ptr()
        del mine
        taken = torch.full((4096,), 7, dtype=torch.uint8, device="cuda")        # (what the allocator hands out next is not the block that the graph still uses)
        assert taken.data_ptr() != address
        assert torch.equal(torch.autograd.grad(loss, h)[0], want)
        assert dev not in ops._scratch                                          # nothing has asked for the shared one
    finally:
        ops._scratch[dev] = shared
        _lib.ext().set_scratch(dev, shared.data_ptr(), shared.numel())
    assert torch.equal(torch.autograd.grad(ops.linear_cross_entropy(h, w, t), h)[0], want)


def test_private_scratch_without_room_for_the_header_is_refused():
    """An expired wait would set a status word behind its end."""
    from nanoquant_b200 import ops

    h = torch.randn((3, 64), device="cuda").bfloat16()
    w = torch.randn((100, 64), device="cuda").bfloat16()
    q, s = ops.quantize_int8(w)
    with ops.private_scratch(torch.zeros(64, dtype=torch.uint8, device="cuda")):
        with pytest.raises(RuntimeError, match="too small"):
            ops.int8_linear_forward(h, q, s)
        with pytest.raises(RuntimeError, match="too small"):
            ops.linear_cross_entropy(h, w, torch.arange(3, device="cuda"))
        assert torch.isfinite(ops.rms_norm(h)).all()        # (needs none)


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
