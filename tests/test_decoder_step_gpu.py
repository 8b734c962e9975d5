"""The calls between a decoder layer's projections as they are used together: quantised q/k/v projections in one launch group, head norms, rotation, cache and attention for prompts,
pieces of prompts and single tokens; captured, compiled, traced, on several streams and behind kernels that release the next one early."""
import threading

import pytest
import torch

from tests.attention_util import attention64, check_attention, check_turned, rand, turned
from tests.util import make_layer, tiles_on_gpu

pytestmark = pytest.mark.gpu

H, K, D, N, R, PAGE = 8, 2, 64, 512, 128, 16


class Layer:
    """Quantised projections of N columns to H query and K key and value heads, head norms, a cache."""

    def __init__(self, seqs, pages, seed=0):
        self.dtype = torch.bfloat16
        self.lin = []
        for i, m in enumerate((H * D, K * D, K * D)):
            L = make_layer(N, R, m, 1, self.dtype, seed=seed + i)
            self.lin.append((L["s_pre"], tiles_on_gpu(L["V"]), L["s_mid"], tiles_on_gpu(L["U"]), L["s_post"], R))
        self.wq, self.wk = (1 + 0.1 * rand(seed + 7, D)), (1 + 0.1 * rand(seed + 8, D))
        self.freq = 1e4 ** (torch.arange(0, D, 2, device="cuda").float() / -D)
        self.cache = [torch.full((seqs * pages + 1, PAGE, K, D), float("nan"), dtype=self.dtype, device="cuda") for _ in range(2)]
        self.table = torch.randperm(seqs * pages + 1, generator=torch.Generator().manual_seed(seed))[:seqs * pages].view(seqs, pages).int().cuda()

    def project(self, x):
        from nanoquant_b200 import ops

        T = len(x)
        scale = 3.0                                               # (outputs of the random factors are small)
        q, k, v = ops.group_forward([x * scale] * 3, self.lin, T, self.dtype, x.device)
        return q.view(T, H, D), k.view(T, K, D), v.view(T, K, D)

    def store(self, q, k, v, positions, sequences=None):
        from nanoquant_b200 import ops

        return ops.append_kv(k, v, *self.cache, self.table, positions, sequences, self.freq, self.wk, q=q, q_weight=self.wq)


def starts(lengths):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device="cuda")


def test_prompts_pieces_and_decoding():
    """Three sequences: their prompts at once, a second piece of two of them, then tokens one by one; every attention against the definition over all keys and values so far, as
    they were projected, normed and rotated to bf16 (which is what the cache holds)."""
    from nanoquant_b200 import ops

    layer = Layer(3, 20)
    lengths = [0, 0, 0]
    kept = [[[], []] for _ in range(3)]

    def run(new, seed):
        x = rand(seed, sum(new), N, dtype=torch.bfloat16)
        q, k, v = layer.project(x)
        seqs = torch.tensor([s for s, n in enumerate(new) for _ in range(n)], dtype=torch.int32, device="cuda")
        pos = torch.tensor([lengths[s] + i for s, n in enumerate(new) for i in range(n)], device="cuda")
        turned_q = layer.store(q, k, v, pos, seqs)
        check_turned(turned_q, *turned(q, pos, layer.freq, layer.wq))
        fresh_q, fresh_k = ops.qk_norm_rope(q, k, pos, layer.freq, layer.wq, layer.wk)
        assert torch.equal(fresh_q, turned_q)
        at = 0
        for s, n in enumerate(new):
            kept[s][0].append(fresh_k[at:at + n])
            kept[s][1].append(v[at:at + n])
            lengths[s] += n
            at += n
        want, at = [], 0
        for s, n in enumerate(new):
            place = torch.arange(lengths[s] - n, lengths[s], device="cuda")
            want.append(attention64(turned_q[at:at + n], torch.cat(kept[s][0]), torch.cat(kept[s][1]), place))
            at += n
        want = [torch.cat([w[i] for w in want]) for i in range(3)]
        table, now = layer.table, torch.tensor(lengths, dtype=torch.int32, device="cuda")
        check_attention(ops.prompt_attention(turned_q, *layer.cache, starts(new), block_table=table, lengths=now), want, new)
        if all(n == l for n, l in zip(new, lengths)):
            check_attention(ops.prompt_attention(turned_q, fresh_k, v, starts(new)), want, new)
        if new == [1, 1, 1]:
            check_attention(ops.paged_attention(turned_q, *layer.cache, table, now), want, new)

    run([37, 150, 1], 1)
    run([90, 0, 33], 2)
    for i in range(20):
        run([1, 1, 1], 10 + i)


def test_decode_step_in_a_graph():
    """One captured step, replayed over positions and lengths that the step itself moves on, from a page into the next; against eager calls on a cache of their own."""
    from nanoquant_b200 import ops

    a, b = Layer(4, 8, seed=3), Layer(4, 8, seed=3)
    begin = [15, 0, 40, 100]
    prompts = rand(5, sum(begin), N, dtype=torch.bfloat16)
    for layer in (a, b):
        seqs = torch.tensor([s for s, n in enumerate(begin) for _ in range(n)], dtype=torch.int32, device="cuda")
        pos = torch.tensor([i for n in begin for i in range(n)], device="cuda")
        layer.store(*layer.project(prompts), pos, seqs)
    x = rand(6, 4, N, dtype=torch.bfloat16)
    pos = torch.tensor(begin, dtype=torch.int32, device="cuda")
    n = torch.zeros_like(pos)

    def step(layer, x, pos, n):
        q = layer.store(*layer.project(x), pos)
        torch.add(pos, 1, out=n)
        o = ops.paged_attention(q, *layer.cache, layer.table, n)
        pos += 1
        return o

    keep_x, keep_pos = x.clone(), pos.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a, x, pos.clone(), n)                                # (warm-up; stores what the first replay stores again)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a, x, pos, n)
    pos.copy_(keep_pos)
    for i in range(25):
        x.copy_(rand(50 + i, 4, N, dtype=torch.bfloat16))
        graph.replay()
        want = step(b, x.clone(), keep_pos, torch.zeros_like(n))
        assert torch.equal(out, want), i
    assert torch.equal(pos, keep_pos)


def test_padded_rows_of_a_captured_batch():
    """A batch captured for more sequences than there are: padded rows store nothing and come back as zeros, whatever their tables say."""
    from nanoquant_b200 import ops

    layer = Layer(4, 6, seed=4)
    layer.table[2:] = -1
    x = rand(7, 4, N, dtype=torch.bfloat16)
    pos = torch.tensor([0, 20, -1, -1], device="cuda")
    before = [c.clone() for c in layer.cache]
    q = layer.store(*layer.project(x), pos)
    assert (q[2:] == 0).all()
    touched = [~((c == b) | (torch.isnan(c) & torch.isnan(b))).all(-1).all(-1) for c, b in zip(layer.cache, before)]
    assert all(t.sum() == 2 for t in touched)
    n = torch.tensor([1, 0, 0, -3], dtype=torch.int32, device="cuda")
    o = ops.paged_attention(q, *layer.cache, layer.table, n)
    assert torch.isfinite(o[0]).all() and (o[1:] == 0).all()


def calls():
    """name -> function of a few tensors that returns tensors."""
    from nanoquant_b200 import ops

    layer = Layer(3, 12, seed=8)
    layer.store(*layer.project(rand(9, 150, N, dtype=torch.bfloat16)), torch.arange(150, device="cuda") % 50,
                (torch.arange(150, device="cuda") // 50).int())
    pos, n = torch.tensor([50, 50, 50], device="cuda"), torch.tensor([51, 30, 7], dtype=torch.int32, device="cuda")
    cu = starts([20, 7, 30])
    qkv = rand(10, 57, H + 2 * K, D, dtype=torch.bfloat16)
    long_table = layer.table.repeat(1, 8)                         # (a width that splits the sequences over the SMs)
    k, v = qkv[:3, H:H + K], qkv[:3, H + K:]

    def append(q):
        cache = [c.clone() for c in layer.cache]
        r = ops.append_kv(k, v, *cache, layer.table, pos, None, layer.freq, layer.wk, q=q, q_weight=layer.wq)
        return r, cache[0][layer.table.long(), 2 + 0 * layer.table.long()], cache[1].nan_to_num()

    return {
        "rope": (qkv[:, :H], lambda q: ops.qk_norm_rope(q, q[:, :2], torch.arange(57, device="cuda"), layer.freq, layer.wq, layer.wk)),
        "append": (qkv[:3, :H], append),
        "paged": (qkv[:3, :H], lambda q: ops.paged_attention(q, *layer.cache, layer.table, n)),
        "paged_split": (qkv[:3, :H], lambda q: ops.paged_attention(q, *layer.cache, long_table, n, window=20)),
        "prompt": (qkv[:, :H], lambda q: ops.prompt_attention(q, qkv[:, H:H + K], qkv[:, H + K:], cu, scale=0.1)),
        "prompt_paged": (qkv[:57, :H], lambda q: ops.prompt_attention(q, *layer.cache, cu, block_table=layer.table, lengths=n, causal=True)),
    }


NAMES = ["rope", "append", "paged", "paged_split", "prompt", "prompt_paged"]


def same(got, want):
    if not isinstance(want, tuple):
        got, want = (got,), (want,)
    return all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) and a.shape == b.shape for a, b in zip(got, want))


@pytest.mark.parametrize("name", NAMES)
def test_trace_records_the_call(name):
    x, fn = calls()[name]
    with torch.no_grad():
        traced = torch.jit.trace(fn, (x,), check_trace=False)
        for y in (x, x * 1.5):
            assert same(traced(y), fn(y))


@pytest.mark.parametrize("name", NAMES)
def test_one_graph_under_torch_compile(name):
    x, fn = calls()[name]
    torch._dynamo.reset()
    with torch.no_grad():
        compiled = torch.compile(fn, fullgraph=True, backend="aot_eager")
        for y in (x, x * 1.5, x):
            assert same(compiled(y), fn(y))


def test_refusals_under_torch_compile():
    from nanoquant_b200 import ops

    x, _ = calls()["rope"]
    f = torch.ones(32, device="cuda")
    pos = torch.arange(57, device="cuda")
    for bad in (lambda q: ops.qk_norm_rope(q.float(), q, pos, f), lambda q: ops.qk_norm_rope(q, q, pos[:3], f), lambda q: ops.prompt_attention(q, q[:, :3], q[:, :3], starts([57]))):
        torch._dynamo.reset()
        with pytest.raises(Exception):
            torch.compile(bad, fullgraph=True, backend="aot_eager")(x)


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_and_subclasses_are_refused(name):
    import torch.autograd.forward_ad as fwad

    x, fn = calls()[name]
    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="forward"):
            fn(fwad.make_dual(x, torch.ones_like(x)))

    class Mine(torch.Tensor):
        pass

    with pytest.raises(RuntimeError, match="plain CUDA tensors"):
        fn(x.as_subclass(Mine))
    fn(x)


def test_registrations_of_the_operators():
    from nanoquant_b200 import ops  # noqa: F401

    op = torch.ops.nanoquant_b200
    layer = Layer(2, 3)
    for c in layer.cache:
        c.zero_()
    q, k = rand(0, 2, H, D, dtype=torch.bfloat16), rand(1, 2, K, D, dtype=torch.bfloat16)
    pos, n, cu = torch.tensor([3, 20], device="cuda"), torch.tensor([4, 21], dtype=torch.int32, device="cuda"), starts([1, 1])
    for f, args in ((op.qk_norm_rope, (q, k, pos, layer.freq, layer.wq, None, 1e-6, False, 1.0)),
                    (op.append_kv, (q, k, k, *layer.cache, layer.table, pos, None, layer.freq, layer.wq, layer.wk, 1e-6, True, 1.0)),
                    (op.append_kv, (None, k, k, *layer.cache, layer.table, pos, None, None, None, None, 1e-6, False, 1.0)),
                    (op.paged_attention, (q, *layer.cache, layer.table, n, 0.125, 0)), (op.prompt_attention, (q, k, k, cu, None, None, None, True, 0.125, 0)),
                    (op.prompt_attention, (q, *layer.cache, cu, None, layer.table, n, False, 0.125, 7))):
        torch.library.opcheck(f.default, args, test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_dynamic"))


def test_two_captured_graphs_at_once():
    """Two graphs on two streams, each with calls that leave partial sums in memory: neither sees the other's."""
    from nanoquant_b200 import ops

    T, total = 40, 3000
    graphs = []
    for seed in range(2):
        k, v = rand(seed, total, K, D, dtype=torch.bfloat16), rand(seed + 2, total, K, D, dtype=torch.bfloat16)
        kc, vc = (t.view(total // 8, 8, K, D) for t in (k, v))
        table = torch.arange(total // 8, dtype=torch.int32, device="cuda")[None]
        q, one = rand(seed + 4, T, H, D, dtype=torch.bfloat16), rand(seed + 6, 1, H, D, dtype=torch.bfloat16)
        n, cu = torch.tensor([total - 5], dtype=torch.int32, device="cuda"), starts([T])

        def run(q=q, one=one, kc=kc, vc=vc, table=table, n=n, cu=cu):
            return ops.prompt_attention(q, kc, vc, cu, block_table=table, lengths=n), ops.paged_attention(one, kc, vc, table, n)

        want = run()
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = [run() for _ in range(4)]
        graphs.append((g, out, want, stream, run))       # (which holds the inputs)
    for _ in range(30):
        for g, _, _, stream, _ in graphs:
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for _, out, want, _, _ in graphs:
        assert all(torch.equal(a, b) for o in out for a, b in zip(o, want))


def test_calls_of_two_threads():
    from nanoquant_b200 import ops

    fns = calls()
    want = {k: fn(x) for k, (x, fn) in fns.items()}
    torch.cuda.synchronize()
    errors, gate = [], threading.Barrier(2)

    def work(order):
        stream = torch.cuda.Stream()
        gate.wait()
        try:
            with torch.cuda.stream(stream), torch.no_grad():
                for i in range(60):
                    name = order[i % len(order)]
                    x, fn = fns[name]
                    got = fn(x)
                    stream.synchronize()
                    if not same(got, want[name]):
                        errors.append(name)
        except Exception as e:  # noqa: BLE001
            errors.append(repr(e))

    threads = [threading.Thread(target=work, args=(o,)) for o in (NAMES, NAMES[::-1])]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors[:3]
    assert ops is not None


@pytest.mark.parametrize("T", [1, 6, 40, 600])
def test_behind_kernels_that_release_the_next_one_early(T):
    """A quantised linear starts the kernel behind it before its outputs are written.  The same buffers again and again with other values: each step has to give what it gives
    with everything complete before every call."""
    from nanoquant_b200 import ops

    layer = Layer(2, 40, seed=5)
    for c in layer.cache:
        c.zero_()
    pos, seqs = torch.arange(T, device="cuda"), torch.ones(T, dtype=torch.int32, device="cuda")
    n, lens, cu = torch.tensor([0, T], dtype=torch.int32, device="cuda"), torch.full((T,), T, dtype=torch.int32, device="cuda"), starts([T])
    xs = [rand(20 + i, T, N, dtype=torch.bfloat16) for i in range(4)]

    def step(x, wait):
        out = []
        pause = torch.cuda.synchronize if wait else lambda: None
        for kind in range(3):
            q, k, v = layer.project(x)
            pause()
            if kind == 0:
                out += ops.qk_norm_rope(q, k, pos, layer.freq, layer.wq, layer.wk)
            elif kind == 1:
                out.append(ops.prompt_attention(q, k, v, cu))
            else:
                q = layer.store(q, k, v, pos, seqs)
                pause()
                out.append(ops.prompt_attention(q, *layer.cache, starts([0, T]), block_table=layer.table, lengths=n))
                out.append(ops.paged_attention(q, *layer.cache, layer.table[1:].expand(T, -1), lens))
                pause()
        return [t.clone() for t in out]

    want = [step(x, True) for x in xs]
    for _ in range(8):
        for x, w in zip(xs, want):
            assert all(torch.equal(a, b) for a, b in zip(step(x, False), w))


def test_wait_that_runs_out():
    """With a limit of one attempt after the first the warps that wait for a long block's end give up: the launch ends, reports, and the next one is right."""
    from nanoquant_b200 import _lib, ops

    L = _lib.lib()
    q, k, v = (rand(s, 2000, 4, 64, dtype=torch.bfloat16) for s in range(3))
    cu = starts([2000])
    want = ops.prompt_attention(q, k, v, cu)
    scratch = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    status = lambda: L.nq_scratch_status(scratch.data_ptr(), torch.cuda.current_stream().cuda_stream)
    with ops.private_scratch(scratch):
        assert torch.equal(ops.prompt_attention(q, k, v, cu), want) and status() == 0
        old = L.nq_gemm_set_wait_limit(1)
        try:
            ops.prompt_attention(q, k, v, cu)
            assert status() == _lib.NQ_ERR_TIMEOUT
        finally:
            assert L.nq_gemm_set_wait_limit(old) == 1
        scratch.zero_()
        assert torch.equal(ops.prompt_attention(q, k, v, cu), want) and status() == 0


@pytest.mark.parametrize("how", ["eager", "compile", "trace"])
def test_calls_without_tokens(how):
    """A decode step, or a batch of prompts, of no sequences: its table has no rows, with or without columns."""
    from nanoquant_b200 import ops

    q, k, v = (rand(i, 3, n, D, dtype=torch.bfloat16)[:0] for i, n in ((0, H), (1, K), (2, K)))
    cache = [torch.zeros((4, PAGE, K, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    freq = 1e4 ** (torch.arange(0, D, 2, device="cuda").float() / -D)
    for columns in (5, 0):
        table = torch.zeros((0, columns), dtype=torch.int32, device="cuda")

        def step(q, k, v, table, none):
            turned_q = ops.append_kv(k, v, *cache, table, none, None, freq, q=q)
            fresh_q, fresh_k = ops.qk_norm_rope(q, k, none, freq)
            start = torch.zeros(2, dtype=torch.int32, device="cuda")
            return turned_q, fresh_q, fresh_k, ops.paged_attention(turned_q, *cache, table, none), ops.prompt_attention(fresh_q, fresh_k, v, start)

        run = {"eager": step, "compile": torch.compile(step, backend="aot_eager", fullgraph=True), "trace": step if how != "trace" else torch.jit.trace(step, (q, k, v, table, none), check_trace=False)}[how]
        got = run(q, k, v, table, none)
        assert [t.shape[0] for t in got] == [0] * 5 and [t.shape[1:] for t in got] == [(H, D), (H, D), (K, D), (H, D), (H, D)]
        assert all((c == 0).all() for c in cache)
    # what is wrong with a call is said without tokens too
    with pytest.raises(RuntimeError, match="lengths"):
        ops.paged_attention(q, *cache, table, none.long())
    with pytest.raises(RuntimeError, match="block_table"):
        ops.paged_attention(q, *cache, torch.zeros((2, 0), dtype=torch.int32, device="cuda"), none)
    with pytest.raises(RuntimeError, match="block_table"):
        ops.append_kv(rand(1, 3, K, D, dtype=torch.bfloat16), rand(2, 3, K, D, dtype=torch.bfloat16), *cache, table, torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="no multiple"):
        ops.paged_attention(q[:, :7], *cache, table, none)


@pytest.mark.parametrize("name", NAMES)
def test_vmap_is_refused(name):
    x, fn = calls()[name]
    with pytest.raises(RuntimeError):
        torch.func.vmap(fn)(torch.stack((x, x)))
