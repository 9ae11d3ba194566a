"""CPU checks of the C ABI: the library loads, exports every declared symbol, and the
ctypes mirrors of the ABI structs have the C layout.  No GPU work is launched."""
import ctypes as C
import os
import re

import pytest

from polar_pack_amd import _native as nat

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "polar_pack.h")


def declared_functions():
    text = open(HEADER).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"^\s*(?:const\s+)?[\w]+\**\s+\**(pp_\w+)\s*\(", text, flags=re.M)))


def test_header_declares_expected_entry_points():
    names = declared_functions()
    for must in ("pp_quad_gemm", "pp_quad_dequant", "pp_quad_stream", "pp_dual_gemm", "pp_dual_dequant",
                 "pp_last_error"):
        assert must in names


def test_library_exports_every_declared_symbol():
    lib = nat.lib()
    missing = [n for n in declared_functions() if not hasattr(lib, n)]
    assert not missing, missing
    # and the binding table covers them all
    assert set(declared_functions()) <= set(nat.EXPORTS)


def test_struct_layouts_match():
    out = (C.c_int64 * 4)()
    assert nat.lib().pp_abi_sizes(out, 4) == 4
    assert out[0] == C.sizeof(nat.QuadProj)
    assert out[1] == C.sizeof(nat.QuadItem)
    assert out[2] == C.sizeof(nat.QuadSeg)
    assert out[3] == C.sizeof(nat.DualProj)


def test_version_and_error_string():
    lib = nat.lib()
    assert b"gfx950" in lib.pp_version()
    assert isinstance(lib.pp_last_error(), bytes)


def test_invalid_arguments_are_rejected_without_a_gpu():
    lib = nat.lib()
    # null LUT array -> PP_EINVAL before any device call
    rc = lib.pp_quad_gemm(None, 0, 0, None, 0, 0, None, 0, None, None, None, 0, 0, None, 0, 0, 1, 1, 1,
                          None, 0, None)
    assert rc == nat.PP_EINVAL
    assert b"luts" in lib.pp_last_error()
    rc = lib.pp_dual_gemm(None, 0, 0, None, 7, 0, 0, None, 32, 0, None, 64, None, None, 1024, 0, None, None, 0, 0,
                          None, None, 0, 0, 1, 1, 1, None, 0, None)
    assert rc == nat.PP_EINVAL
    assert b"code_layout" in lib.pp_last_error()
    with pytest.raises(RuntimeError):
        nat.check(rc, "pp_dual_gemm")


def test_stream_rows_query():
    assert nat.lib().pp_quad_stream_rows(1) >= 1
    assert nat.lib().pp_quad_stream_rows(9) == 0
    assert b"1..8" in nat.lib().pp_last_error()


def test_cache_layout_matches():
    out = (C.c_int64 * 5)()
    assert nat.lib().pp_abi_sizes(out, 5) == 5
    assert out[4] == C.sizeof(nat.KVCache)
    # the fields where the header has them: four addresses, 64-bit pages, four 32-bit sizes
    assert [getattr(nat.KVCache, f).offset for f, _ in nat.KVCache._fields_] == [0, 8, 16, 24, 32, 40, 44, 48, 52]


CACHE = dict(k=4096, v=8192, k_scale=64, v_scale=64, pages=4, heads=2, head_dim=64, block=16, codes=nat.PP_KV_INT8)
SEQS = dict(table=64, ld=3, width=3, lengths=64, cu=64, batch=2)


def calls(cache, seqs, dtype=nat.PP_F16, tokens=5, q_heads=4, window=0, causal=1):
    """The status of each cache entry point for these descriptions: with null operands all are refused, here or at the end,
    before any device call."""
    lib, c = nat.lib(), nat.KVCache(**cache)
    s = [seqs[k] for k in ("table", "ld", "width", "lengths", "cu", "batch")]
    at = C.addressof(c)
    append = lib.pp_kv_append(at, None, 128, 64, None, 128, 64, dtype, tokens, *s, None)
    read = lib.pp_kv_read(at, *s, tokens, dtype, None, None, None)
    attend = lib.pp_kv_attention(at, None, 256, 64, q_heads, dtype, tokens, *s, causal, window, 0.125, None, None, None,
                                 0, None, 0, None)
    return append, read, attend


@pytest.mark.parametrize("change,word", [
    (dict(k=None), b"null"), (dict(pages=0), b"pages"), (dict(pages=2 ** 31), b"pages"), (dict(heads=0), b"heads"),
    (dict(block=48), b"block"), (dict(head_dim=80), b"head_dim"), (dict(codes=7), b"codes"), (dict(v=4100), b"aligned")])
def test_caches_that_are_refused(change, word):
    assert calls({**CACHE, **change}, SEQS) == (nat.PP_EINVAL,) * 3
    assert word in nat.lib().pp_last_error()


@pytest.mark.parametrize("change,word", [
    (dict(table=None), b"null"), (dict(lengths=None), b"null"), (dict(batch=0), b"batch"), (dict(width=0), b"block table"),
    (dict(width=2 ** 27, ld=2 ** 27), b"block table"), (dict(ld=2), b"overlap"), (dict(cu=None), b"cu")])
def test_sequences_that_are_refused(change, word):
    assert calls(CACHE, {**SEQS, **change}) == (nat.PP_EINVAL,) * 3
    assert word in nat.lib().pp_last_error()


def test_serving_calls_that_are_refused():
    lib = nat.lib()
    no = nat.PP_EINVAL
    assert calls(CACHE, SEQS, tokens=-1) == (no,) * 3
    assert calls(CACHE, SEQS, tokens=2 ** 28 + 1) == (no,) * 3
    assert calls(CACHE, SEQS, dtype=9) == (no,) * 3
    assert calls(CACHE, SEQS, dtype=nat.PP_F32)[::2] == (no, no)        # values are 16 bits
    assert calls(CACHE, SEQS, q_heads=5)[2] == no and b"query heads" in lib.pp_last_error()
    assert calls(CACHE, SEQS, window=-1)[2] == no and calls(CACHE, SEQS, window=3, causal=0)[2] == no
    assert calls(CACHE, SEQS) == (no,) * 3                              # null keys, outputs, queries
    assert lib.pp_kv_append(None, None, 128, 64, None, 128, 64, nat.PP_F16, 5, 64, 3, 3, 64, 64, 2, None) == no

    def logprobs(x=64, dtype=nat.PP_F32, rows=2, V=100, tokens=64, per_row=1, top=0, out=64, entropy=64, ids=None,
                 lps=None):
        return lib.pp_logprobs(x, V, dtype, rows, V, tokens, per_row, per_row, top, out, entropy, ids, lps, None, 0, None)
    for bad in (dict(dtype=9), dict(rows=-1), dict(rows=2 ** 24 + 1), dict(V=0), dict(V=2 ** 30 + 1), dict(top=-1),
                dict(top=65), dict(top=101, V=100), dict(per_row=-1), dict(x=None), dict(x=66), dict(entropy=None),
                dict(tokens=None), dict(out=None), dict(top=5)):
        assert logprobs(**bad) == no, bad
        assert b"pp_logprobs" in lib.pp_last_error()
    assert logprobs(rows=0) == nat.PP_OK


def test_serving_sizes_of_nothing():
    lib = nat.lib()
    assert lib.pp_kv_attention_workspace_size(2, 64, 16, 3, 2, 0, 4) == 0
    assert lib.pp_kv_attention_counts_size(2, 64, 16, 3, 0, 5, 4) == 0
    assert lib.pp_logprobs_workspace_size(0, 100, 5) == 0
