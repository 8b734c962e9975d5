"""CPU-only: addresses that an operand's elements cannot have are refused by the C ABI of the norms, the 8-bit linear and the loss (before any CUDA call): the
kernels' loads would fault."""
import os

import pytest

from nanoquant_b200 import _lib

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built (python -m nanoquant_b200.build)")
P = 0x10000                        # never read
F16, F32 = _lib.NQ_F16, _lib.NQ_F32


def refused(name, good, at):
    """`at`: index of a pointer -> the multiple its address has to be."""
    fn = getattr(_lib.lib(), name)
    for i, multiple in at.items():
        a = list(good)
        a[i] = P + multiple // 2
        assert fn(*a) == _lib.NQ_ERR_ALIGN, (name, i)


def test_addresses():
    L = _lib.lib()
    refused("nq_norm_fwd", [P, P, P, P, P, 4, 64, 64, 64, 1e-5, 1, F16, F16, None], {0: 2, 1: 2, 2: 2, 3: 2, 4: 8})
    refused("nq_norm_fwd", [P, P, P, P, P, 4, 64, 64, 64, 1e-5, 1, F16, F32, None], {0: 2, 1: 4, 2: 4, 3: 2, 4: 8})
    need = L.nq_norm_bwd_scratch_bytes(4, 64)
    refused("nq_norm_bwd", [P, P, P, P, P, P, P, P, need, 4, 64, 64, 64, 64, 1, F16, F16, None], {0: 2, 1: 2, 2: 2, 3: 8, 4: 2, 5: 2, 6: 2, 7: 16})
    refused("nq_norm_bwd", [P, P, P, P, P, P, P, P, need, 4, 64, 64, 64, 64, 1, F16, F32, None], {2: 4, 5: 4, 6: 4})
    refused("nq_quantize_rows_s8", [P, P, P, 4, 64, 64, 64, F16, None], {0: 2, 2: 4})
    need = L.nq_int8_linear_scratch_bytes(30, 100)
    refused("nq_int8_linear_fwd", [P, P, P, P, P, P, need, P, 30, 100, 50, 100, 112, 50, F16, None], {0: 2, 1: 16, 2: 16, 3: 2, 4: 2, 5: 16, 7: 16})
    for bits in (32, 64):
        need = L.nq_linear_ce_fwd_scratch_bytes(5, 64, 100)
        refused("nq_linear_ce_fwd", [P, P, P, bits, -100, P, P, P, P, need, P, 5, 64, 100, 64, 64, 2, F16, None], {0: 16, 1: 16, 2: bits // 8, 5: 4, 6: 4, 7: 4, 8: 16, 10: 16})
        need = L.nq_linear_ce_bwd_scratch_bytes(5, 64, 100)
        refused("nq_linear_ce_bwd", [P, P, P, bits, -100, P, P, P, 0, P, P, P, need, P, 5, 64, 100, 64, 64, 64, 64, 0, F16, None],
                {0: 16, 1: 16, 2: bits // 8, 5: 4, 6: 4, 7: 4, 9: 16, 10: 16, 11: 16, 13: 16})
