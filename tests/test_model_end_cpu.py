"""CPU-only: what the C ABI of the norms, the 8-bit linear and the loss refuses (before any CUDA call), and the sizes it reports."""
import os

import pytest

from nanoquant_b200 import _lib

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built (python -m nanoquant_b200.build)")
P, ODD = 0x10000, 0x10002          # addresses that are never read
F16, BF16, F32 = _lib.NQ_F16, _lib.NQ_BF16, _lib.NQ_F32


def call(name, good, index, value):
    a = list(good)
    a[index] = value
    return getattr(_lib.lib(), name)(*a)


def test_norm_forward_refusals():
    good = [P, P, P, P, P, 4, 64, 64, 64, 1e-5, 1, F16, F16, None]     # x w b y stats rows N ldx ldy eps center dtype weight_dtype stream
    for i, v, st in ((0, None, "NULL"), (3, None, "NULL"), (5, 0, "SHAPE"), (6, 0, "SHAPE"), (7, -1, "SHAPE"), (8, 63, "SHAPE"), (11, F32, "DTYPE"), (11, 7, "DTYPE"),
                     (12, BF16, "DTYPE"), (6, 20000, "SHAPE"), (5, 1 << 31, "TOO_LARGE")):
        assert call("nq_norm_fwd", good, i, v) == getattr(_lib, "NQ_ERR_" + st), (i, v)
    big = _lib.lib().nq_norm_max_columns() + 1
    assert _lib.lib().nq_norm_fwd(P, P, P, P, P, 4, big, big, big, 1e-5, 1, F16, F16, None) == _lib.NQ_ERR_TOO_LARGE


def test_norm_backward_refusals():
    L = _lib.lib()
    need = L.nq_norm_bwd_scratch_bytes(4, 64)
    assert need >= 2 * 4 * 64 * 4 and L.nq_norm_bwd_scratch_bytes(0, 64) == 0
    assert L.nq_norm_bwd_scratch_bytes(10 ** 6, 64) <= 8 * 200 * 2 * 64 * 4            # by CTAs, not by rows
    good = [P, P, P, P, P, P, P, P, need, 4, 64, 64, 64, 64, 1, F16, F16, None]   # dy x w stats dx dw db scratch bytes rows N lddy ldx lddx ...
    for i, v, st in ((0, None, "NULL"), (1, None, "NULL"), (3, None, "NULL"), (7, None, "NULL"), (7, ODD, "ALIGN"), (8, need - 1, "SCRATCH"), (9, 0, "SHAPE"),
                     (13, 63, "SHAPE"), (15, F32, "DTYPE"), (16, BF16, "DTYPE")):
        assert call("nq_norm_bwd", good, i, v) == getattr(_lib, "NQ_ERR_" + st), (i, v)
    nothing = list(good)
    nothing[4:7] = [None] * 3
    assert L.nq_norm_bwd(*nothing) == _lib.NQ_OK


def test_int8_refusals():
    L = _lib.lib()
    good = [P, P, P, 4, 64, 64, 64, F16, None]                          # x q scale rows N ldx ldq dtype stream
    for i, v, st in ((0, None, "NULL"), (1, None, "NULL"), (2, None, "NULL"), (3, 0, "SHAPE"), (4, 0, "SHAPE"), (6, 63, "SHAPE"), (7, F32, "DTYPE"),
                     (3, 1 << 31, "TOO_LARGE")):
        assert call("nq_quantize_rows_s8", good, i, v) == getattr(_lib, "NQ_ERR_" + st), (i, v)
    need = L.nq_int8_linear_scratch_bytes(30, 100)
    assert need == 256 + 30 * 112 and L.nq_int8_linear_scratch_bytes(0, 8) == 0 and L.nq_int8_linear_scratch_bytes(1, 4096) == 0
    good = [P, P, P, P, P, P, need, P, 30, 100, 50, 100, 112, 50, BF16, None]   # x w ws bias y scratch bytes status T N V ldx ldw ldy dtype stream
    for i, v, st in ((0, None, "NULL"), (1, None, "NULL"), (2, None, "NULL"), (4, None, "NULL"), (5, None, "NULL"), (7, None, "NULL"), (6, need - 1, "SCRATCH"),
                     (1, ODD, "ALIGN"), (2, ODD, "ALIGN"), (5, ODD, "ALIGN"), (7, ODD, "ALIGN"), (8, 0, "SHAPE"), (9, 0, "SHAPE"), (10, 0, "SHAPE"), (12, 96, "SHAPE"),
                     (12, 120, "SHAPE"), (13, 49, "SHAPE"), (14, F32, "DTYPE"), (10, 1 << 30, "SHAPE")):
        assert call("nq_int8_linear_fwd", good, i, v) == getattr(_lib, "NQ_ERR_" + st), (i, v)
    wide = list(good)
    wide[9], wide[11], wide[12] = 131073, 131073, 131088
    assert L.nq_int8_linear_fwd(*wide) == _lib.NQ_ERR_TOO_LARGE


def test_loss_refusals():
    L = _lib.lib()
    T, N, V = 5, 64, 100
    need = L.nq_linear_ce_fwd_scratch_bytes(T, N, V)
    assert need > 0 and L.nq_linear_ce_fwd_scratch_bytes(T, 60, V) == 0 and L.nq_linear_ce_fwd_scratch_bytes(0, N, V) == 0
    # h w targets bits ignore loss lse count scratch bytes status T N V ldh ldw reduction dtype stream
    good = [P, P, P, 64, -100, P, P, P, P, need, P, T, N, V, N, N, 2, BF16, None]
    cases = [(i, None, "NULL") for i in (0, 1, 2, 5, 6, 7, 8, 10)] + [(0, ODD, "ALIGN"), (1, ODD, "ALIGN"), (8, ODD, "ALIGN"), (10, ODD, "ALIGN"), (3, 16, "DTYPE"),
             (9, need - 1, "SCRATCH"), (11, 0, "SHAPE"), (12, 60, "SHAPE"), (13, 0, "SHAPE"), (14, 56, "SHAPE"), (14, 68, "SHAPE"), (15, 56, "SHAPE"),
             (16, 3, "UNSUPPORTED"), (16, -1, "UNSUPPORTED"), (17, F32, "DTYPE"), (11, 1 << 23, "TOO_LARGE"), (13, 1 << 25, "TOO_LARGE")]
    for i, v, st in cases:
        assert call("nq_linear_ce_fwd", good, i, v) == getattr(_lib, "NQ_ERR_" + st), (i, v)
    need = L.nq_linear_ce_bwd_scratch_bytes(T, N, V)
    # h w targets bits ignore lse count grad stride dh dw scratch bytes status T N V ldh ldw lddh lddw reduction dtype stream
    good = [P, P, P, 64, -100, P, P, P, 0, P, P, P, need, P, T, N, V, N, N, N, N, 0, F16, None]
    cases = [(i, None, "NULL") for i in (0, 1, 2, 5, 6, 7, 11, 13)] + [(i, ODD, "ALIGN") for i in (0, 1, 9, 10, 11, 13)] + [
        (3, 8, "DTYPE"), (12, need - 1, "SCRATCH"), (14, 0, "SHAPE"), (19, 56, "SHAPE"), (20, 68, "SHAPE"), (21, 3, "UNSUPPORTED"), (22, F32, "DTYPE")]
    for i, v, st in cases:
        assert call("nq_linear_ce_bwd", good, i, v) == getattr(_lib, "NQ_ERR_" + st), (i, v)
    nothing = list(good)
    nothing[9] = nothing[10] = None
    assert L.nq_linear_ce_bwd(*nothing) == _lib.NQ_OK


@pytest.mark.parametrize("T,N,V", [(1, 4096, 151936), (128, 4096, 151936), (2048, 4096, 151936), (4096, 4096, 32000), (77, 512, 1003), (30000, 64, 151936)])
def test_loss_scratch_is_a_piece_and_not_the_logits(T, N, V):
    """One piece of the vocabulary (256 MB, or 256 words), the hidden states once more and the partial sums of dh (256 MB); forward 8 bytes for every 64 words
    and token of one product, and the hidden states of these."""
    piece = max(256 << 20, T * 256 * 2)
    assert _lib.lib().nq_linear_ce_bwd_scratch_bytes(T, N, V) <= piece + 2 * T * N + 2 * (256 << 20) + 16 * T + 4096
    assert _lib.lib().nq_linear_ce_fwd_scratch_bytes(T, N, V) <= 2 * (V // 64 + 1) * min(T, 16384) * 8 + 2 * min(T, 16384) * N + 16 * T + 2048
