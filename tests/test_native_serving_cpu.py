"""CPU checks of the C entries of the 4-bit cache, the append with the rotation and the drafts: what they refuse, before
any device call."""
import ctypes as C

import pytest

from polar_pack_amd import _native as nat

NO = nat.PP_EINVAL
CACHE = dict(k=4096, v=8192, k_scale=4096, v_scale=4096, pages=4, heads=2, head_dim=64, block=16, codes=nat.PP_KV_E2M1)
ROTARY = dict(turns=64, axes=None, rotary_dim=64, n_axes=1, pairs=0, scaling=1.0)
SEQS = (64, 3, 3, 64, 64, 2)


def rotate_append(cache=CACHE, rotary=ROTARY, q=64, q_heads=4, q_out=64, k=64, v=64, dtype=nat.PP_F16, tokens=5, pos=None,
                  pos_type=nat.PP_POS_I64, seqs=SEQS):
    c, r = nat.KVCache(**cache), nat.Rotary(**rotary) if rotary else None
    return nat.lib().pp_kv_rotate_append(C.addressof(c), q, 256, 64, q_heads, q_out, k, 128, 64, v, 128, 64, dtype, tokens,
                                         C.addressof(r) if r else None, pos, 0, pos_type, *seqs, None)


@pytest.mark.parametrize("change", [dict(k=None), dict(k_scale=4100), dict(v_scale=4104), dict(v=8200), dict(block=48),
                                    dict(head_dim=80), dict(codes=3), dict(pages=0), dict(k_scale=None)])
def test_caches_that_are_refused(change):
    c = nat.KVCache(**{**CACHE, **change})
    at, lib = C.addressof(c), nat.lib()
    assert rotate_append({**CACHE, **change}) == NO
    assert lib.pp_kv_append(at, 64, 128, 64, 64, 128, 64, nat.PP_F16, 5, *SEQS, None) == NO
    assert lib.pp_kv_read(at, *SEQS, 5, nat.PP_F16, 64, 64, None) == NO
    assert lib.pp_kv_attention(at, 64, 256, 64, 4, nat.PP_F16, 5, *SEQS, 1, 0, 0.125, 64, None, None, 0, None, 0, None) == NO


@pytest.mark.parametrize("change", [dict(rotary=None), dict(rotary={**ROTARY, "rotary_dim": 80}), dict(rotary={**ROTARY, "turns": None}),
                                    dict(k=None), dict(v=None), dict(k=65), dict(q=None), dict(q_out=None), dict(q_out=72),
                                    dict(q=65), dict(q_heads=-1), dict(q_heads=65536), dict(dtype=nat.PP_F32), dict(tokens=-1),
                                    dict(pos=68), dict(pos_type=2), dict(seqs=(None, *SEQS[1:])), dict(seqs=(64, 2, 3, 64, 64, 2)),
                                    dict(seqs=(64, 3, 3, 64, None, 2))])
@pytest.mark.parametrize("codes", [nat.PP_KV_INT8, nat.PP_KV_E2M1])
def test_turned_appends_that_are_refused(codes, change):
    assert rotate_append({**CACHE, "codes": codes}, **change) == NO
    assert nat.lib().pp_last_error()


def test_no_tokens():
    assert rotate_append(tokens=0) == nat.PP_OK


@pytest.mark.parametrize("change", [dict(dtype=9), dict(batch=-1), dict(batch=2 ** 24 + 1), dict(n=-1), dict(n=2 ** 16 + 1), dict(V=0),
                                    dict(V=2 ** 30 + 1), dict(p=None), dict(p=66), dict(q=65), dict(tokens=None), dict(u=None),
                                    dict(out=None), dict(accepted=None), dict(ws=None), dict(ws=68), dict(size=8), dict(done=None),
                                    dict(done_size=4)])
def test_drafts_that_are_refused(change):
    lib = nat.lib()
    a = {**dict(p=64, q=64, dtype=nat.PP_F32, batch=2, n=3, V=100, tokens=64, u=64, out=64, accepted=64, ws=64, size=1 << 20, done=64,
                done_size=8), **change}

    def call():
        return lib.pp_verify_drafts(a["p"], 400, 100, a["q"], 300, 100, a["dtype"], a["batch"], a["n"], a["V"], a["tokens"], 3, a["u"],
                                    4, None, a["out"], a["accepted"], a["ws"], a["size"], a["done"], a["done_size"], None)
    assert call() == NO
    assert b"pp_verify_drafts" in lib.pp_last_error()


def test_no_sequences():
    assert nat.lib().pp_verify_drafts(None, 0, 0, None, 0, 0, nat.PP_F32, 0, 3, 100, None, 0, None, 0, None, None, None, None, 0, None,
                                      0, None) == nat.PP_OK
    assert nat.lib().pp_verify_drafts_workspace_size(0, 100) == 0
