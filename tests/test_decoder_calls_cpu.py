"""CPU-only: what the C ABI of the calls between a decoder layer's projections refuses (before any CUDA call), the sizes it reports, and the structures that the loader passes."""
import ctypes
import os
import re
import subprocess
import sys

import pytest

from nanoquant_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built (python -m nanoquant_b200.build)")
P = 0x10000                        # an address that is never read
F16, BF16, F32 = _lib.NQ_F16, _lib.NQ_BF16, _lib.NQ_F32


def refused(call, good, cases):
    for field, value, status in cases:
        d = dict(good)
        d.update({field: value} if isinstance(field, str) else dict(zip(field, value)))
        assert call(d) == getattr(_lib, "NQ_ERR_" + status), (field, value)


@pytest.mark.parametrize("name,desc", [("nq_heads_desc", _lib.HeadsDesc), ("nq_attention_desc", _lib.AttentionDesc)])
def test_structures_are_the_headers(name, desc):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "nanoquant_b200.h")).read(), flags=re.S)
    body = [b for b, n in re.findall(r"typedef struct \{([^}]*)\}\s*(\w+);", text) if n == name][0]
    fields = []
    for line in body.split(";"):
        m = re.match(r"\s*(const\s+)?(\w+)\s*(.*)", line.strip(), re.S)
        if not m or not line.strip():
            continue
        for var in m.group(3).split(","):
            var = var.strip()
            kind = ctypes.c_void_p if "*" in line else {"int64_t": ctypes.c_int64, "int": ctypes.c_int, "float": ctypes.c_float}[m.group(2)]
            fields.append((var.replace("*", "").strip(), kind))
    assert fields == list(desc._fields_)


def heads(d):
    return _lib.lib().nq_heads_fwd(ctypes.byref(_lib.HeadsDesc(**d)), None)


HEADS = dict(q=P, k=P, v=P, q_out=P, k_out=P, positions=P, inv_freq=P, q_weight=P, k_weight=P, q_token=512, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64, T=3,
             position_bits=32, q_heads=8, k_heads=2, D=64, R=64, weight_dtype=F16, dtype=F16, eps=1e-6, scaling=1.0)
CACHED = dict(HEADS, k_out=None, k_cache=P, v_cache=P, block_table=P, sequences=P, kc_page=2048, kc_slot=128, kc_head=64, vc_page=2048, vc_slot=128, vc_head=64, table_stride=4, pages=9,
              seqs=2, max_pages=4, page_size=16)


def test_heads_refusals():
    assert _lib.lib().nq_heads_fwd(None, None) == _lib.NQ_ERR_NULL
    refused(heads, HEADS, [(n, None, "NULL") for n in ("q", "k", "q_out", "k_out", "positions", "inv_freq")] + [
        (n, P + 8, "ALIGN") for n in ("q", "k", "v", "q_out", "k_out", "q_weight", "k_weight")] + [("inv_freq", P + 2, "ALIGN"), ("positions", P + 2, "ALIGN"), (("positions", "position_bits"), (P + 4, 64), "ALIGN"),
        ("dtype", F32, "DTYPE"), ("weight_dtype", BF16, "DTYPE"), ("position_bits", 16, "DTYPE"), ("T", 0, "SHAPE"), ("D", 60, "SHAPE"), ("D", 0, "SHAPE"), ("R", 66, "SHAPE"), ("R", 63, "SHAPE"), ("R", -2, "SHAPE"),
        ("q_heads", -1, "SHAPE"), (("q_heads", "k_heads"), (0, 0), "SHAPE"), ("q_head", 65, "SHAPE"), ("k_token", 4, "SHAPE"), ("D", 264, "TOO_LARGE"), ("T", 1 << 31, "TOO_LARGE"), ("q_heads", (1 << 16) + 1, "TOO_LARGE")])
    refused(heads, CACHED, [(n, None, "NULL") for n in ("k_cache", "v_cache", "v", "block_table")] + [(n, P + 8, "ALIGN") for n in ("k_cache", "v_cache")] + [
        ("block_table", P + 1, "ALIGN"), ("sequences", P + 2, "ALIGN"), ("page_size", 24, "SHAPE"), ("page_size", 4, "SHAPE"), ("page_size", 0, "SHAPE"), ("pages", 0, "SHAPE"), ("max_pages", 0, "SHAPE"),
        ("seqs", 0, "SHAPE"), ("table_stride", -1, "SHAPE"), ("kc_slot", 129, "SHAPE"), ("vc_page", 4, "SHAPE"), ("k_heads", 0, "SHAPE")])
    assert _lib.lib().nq_head_max_columns() == 256


PACKED = dict(q=P, k=P, v=P, out=P, cu_seqlens=P, q_token=512, q_head=64, k_slot=128, k_head=64, v_slot=128, v_head=64, T=10, Tk=10, seqs=2, q_heads=8, k_heads=2, D=64, causal=1, dtype=BF16, scale=0.125)
PAGED = dict(PACKED, lengths=P, block_table=P, k_page=2048, v_page=2048, table_stride=40, pages=9, max_pages=40, page_size=16)
COMMON = [(n, None, "NULL") for n in ("q", "k", "v", "out")] + [(n, P + 8, "ALIGN") for n in ("q", "k", "v", "out")] + [
    ("dtype", F32, "DTYPE"), ("seqs", 0, "SHAPE"), ("q_heads", 7, "SHAPE"), ("k_heads", 0, "SHAPE"), ("D", 60, "SHAPE"), ("D", 264, "TOO_LARGE"), ("window", -1, "SHAPE"), ("scale", 0.0, "SHAPE"),
    ("scale", -1.0, "SHAPE"), ("scale", float("nan"), "SHAPE"), ("scale", float("inf"), "SHAPE"), ("q_token", 4, "SHAPE"), ("v_head", 65, "SHAPE")]
CACHE = [("lengths", None, "NULL"), ("lengths", P + 2, "ALIGN"), ("block_table", P + 2, "ALIGN"), ("page_size", 12, "SHAPE"), ("page_size", 4, "SHAPE"), ("pages", 0, "SHAPE"), ("max_pages", 0, "SHAPE"),
         ("k_page", 4, "SHAPE"), ("table_stride", -1, "SHAPE"), ("pages", 1 << 31, "TOO_LARGE")]


def test_paged_attention_refusals():
    L = _lib.lib()
    need = L.nq_paged_attention_scratch_bytes(2, 8, 2, 64, 640)
    assert need > 0 and need % 16 == 0 and L.nq_paged_attention_scratch_bytes(2, 8, 2, 64, 256) == 0 and L.nq_paged_attention_scratch_bytes(0, 8, 2, 64, 640) == 0
    assert L.nq_paged_attention_scratch_bytes(1000, 8, 2, 64, 1 << 20) == need                  # by CTAs, not by sequences
    assert L.nq_paged_attention_fwd(None, P, need, P, None) == _lib.NQ_ERR_NULL
    call = lambda d, scratch=P, n=need, status=P: L.nq_paged_attention_fwd(ctypes.byref(_lib.AttentionDesc(**d)), scratch, n, status, None)
    refused(call, PAGED, COMMON + CACHE + [("block_table", None, "NULL"), (("max_pages", "page_size"), (1 << 20, 1 << 12), "TOO_LARGE")])
    assert call(PAGED, None) == _lib.NQ_ERR_NULL and call(PAGED, P + 4) == _lib.NQ_ERR_ALIGN and call(PAGED, P, need - 1) == _lib.NQ_ERR_SCRATCH
    assert call(PAGED, P, need, None) == _lib.NQ_ERR_NULL and call(PAGED, P, need, P + 4) == _lib.NQ_ERR_ALIGN


def test_prompt_attention_refusals():
    L = _lib.lib()
    call = lambda d, status=P, scratch=None, n=0: L.nq_prompt_attention_fwd(ctypes.byref(_lib.AttentionDesc(**d)), scratch, n, status, None)
    assert L.nq_prompt_attention_fwd(None, None, 0, P, None) == _lib.NQ_ERR_NULL
    more = [("cu_seqlens", None, "NULL"), ("cu_seqlens", P + 2, "ALIGN"), ("T", 0, "SHAPE"), (("q_heads", "k_heads"), (129, 1), "SHAPE"), ("T", 1 << 30, "TOO_LARGE")]
    refused(call, PACKED, COMMON + more + [("Tk", 0, "SHAPE"), ("cu_seqlens_k", P + 2, "ALIGN"), ("Tk", 1 << 30, "TOO_LARGE")])
    refused(call, PAGED, COMMON + more + CACHE + [(("max_pages", "page_size"), (1 << 20, 1 << 10), "TOO_LARGE")])
    assert call(PACKED, None) == _lib.NQ_ERR_NULL and call(PACKED, P + 4) == _lib.NQ_ERR_ALIGN
    size = lambda **kw: L.nq_prompt_attention_scratch_bytes(ctypes.byref(_lib.AttentionDesc(**{**PAGED, **kw})))
    need = size(max_pages=1024)                                   # few tokens behind a long cache: parts of it by several CTAs
    assert need > 0 and need % 16 == 0 and size() == 0 and size(D=60) == 0 and L.nq_prompt_attention_scratch_bytes(None) == 0
    long = dict(PAGED, max_pages=1024)
    assert call(long) == _lib.NQ_ERR_NULL and call(long, P, P + 4, need) == _lib.NQ_ERR_ALIGN and call(long, P, P, need - 1) == _lib.NQ_ERR_SCRATCH
    for kw in (dict(T=100000), dict(T=100), dict(T=1, seqs=1000), dict(q_heads=64, k_heads=64, D=256), dict(q_heads=128, k_heads=1)):
        assert size(max_pages=1 << 16, **kw) < 1 << 28, kw         # whatever the sizes


def test_sequences_in_a_cache_have_up_to_two_to_the_30_tokens():
    """Windows are cut to that, and so are the tables that a window could be too short for."""
    L = _lib.lib()
    d = _lib.AttentionDesc(**{**PAGED, "max_pages": 1 << 26, "table_stride": 1 << 26})
    assert L.nq_paged_attention_fwd(ctypes.byref(d), P, 1 << 40, P, None) == _lib.NQ_ERR_TOO_LARGE
    assert L.nq_prompt_attention_fwd(ctypes.byref(d), P, 1 << 40, P, None) == _lib.NQ_ERR_TOO_LARGE


@pytest.mark.parametrize("sizes", [(1, 1, 2, 128, 1 << 17), (1, 7, 2, 128, 1 << 17), (1, 8, 2, 60, 1 << 17), (1, 8, 2, 264, 1 << 17), (1, 8, 0, 64, 1 << 17), (1, 0, 2, 64, 1 << 17), (1, -8, -2, 64, 1 << 17),
                                   (1, (1 << 16) + 2, 2, 64, 1 << 17), (1 << 30, 8, 2, 64, 1 << 17), (1, 8, 2, 64, 1 << 30), (1, 8, 2, 64, 0), (1, 8, 2, 64, -1 << 20), (-3, 8, 2, 64, 1 << 17)])
def test_paged_attention_asks_for_no_scratch_for_what_it_refuses(sizes):
    """In a process of its own: fewer query heads than key heads ended it (a division by zero)."""
    code = f"from nanoquant_b200 import _lib; print(_lib.lib().nq_paged_attention_scratch_bytes(*{sizes!r}))"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert (r.returncode, r.stdout.strip()) == (0, "0"), (r.returncode, r.stderr[-300:])
