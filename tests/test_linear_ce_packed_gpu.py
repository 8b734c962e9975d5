"""The larger calls of `ops.linear_cross_entropy`, which pack the rows that have a target, in the forms that the small ones are tested in: other types of targets,
other numbers for none, rows apart, one gradient alone.  What these do not change has the same bits."""
import pytest
import torch

from tests.test_linear_ce_gpu import make, run

pytestmark = pytest.mark.gpu

T, N, V = 700, 2048, 80000


@pytest.fixture(scope="module", params=[torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def call(request):
    h, w, t = make(T, N, V, request.param, seed=17, ignored=0.4)
    t[t == 7] = 8
    h[t == -100] = float("nan")
    return h, w, t, run(h, w, t, "mean", 64.0)


@pytest.mark.parametrize("ignore", [-100, 7, -1, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("wide", [True, False])
def test_targets_of_either_type_and_any_number_for_none(call, ignore, wide):
    h, w, t, want = call
    other = torch.where(t == -100, ignore, t)
    got = run(h, w, other if wide else other.int(), "mean", 64.0, ignore_index=ignore)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("off", [8, 3])
def test_rows_apart(call, off):
    h, w, t, want = call
    wide = torch.full((T, N + 24), float("nan"), dtype=h.dtype, device="cuda")
    wide[:, off:off + N] = h
    got = run(wide[:, off:off + N], w, t, "mean", 64.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_one_gradient_alone(call):
    from nanoquant_b200 import ops

    h, w, t, want = call
    g = torch.tensor(64.0, device="cuda")
    for i, leaf in enumerate((h, w)):
        leaf = leaf.detach().requires_grad_()
        loss = ops.linear_cross_entropy(*((leaf, w) if i == 0 else (h, leaf)), t)
        (d,) = torch.autograd.grad(loss, leaf, g)
        assert torch.equal(loss.detach(), want[0]) and torch.equal(d, want[1 + i])


def test_a_graph_used_twice(call):
    """Nothing of a call's scratch is left over from its forward pass: the second backward pass gives the first one's bits."""
    from nanoquant_b200 import ops

    h, w, t, want = call
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = ops.linear_cross_entropy(h, w, t)
    for _ in range(2):
        got = torch.autograd.grad(loss, (h, w), torch.tensor(64.0, device="cuda"), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want[1:]))
        ops.linear_cross_entropy(h.detach().nan_to_num().flip(0).contiguous(), w.detach(), t)       # (another call in between)
