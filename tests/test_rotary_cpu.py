"""What Rotary and rotate refuse before any device is asked, and the C entries' checks."""
import ctypes as C

import pytest
import torch

from polar_pack_amd import _native as nat
from polar_pack_amd.rotary import Rotary


@pytest.mark.parametrize("args", [
    dict(head_dim=60), dict(head_dim=8), dict(head_dim=520), dict(head_dim=64, rotary_dim=24), dict(head_dim=64, rotary_dim=80),
    dict(head_dim=64, rotary_dim=0), dict(head_dim=64, pairs="both"), dict(head_dim=64, base=-1.0),
    dict(head_dim=64, base=float("inf")), dict(head_dim=64, inv_freq=[1.0] * 31), dict(head_dim=64, inv_freq=[float("nan")] * 32),
    dict(head_dim=64, sections=(16, 8)), dict(head_dim=64, sections=(40, -8)), dict(head_dim=64, axes=[0] * 31),
    dict(head_dim=64, axes=[-1] + [0] * 31), dict(head_dim=64, axes=[255] * 32),
    dict(head_dim=64, sections=(16, 16), axes=[0] * 32), dict(head_dim=64, scaling=float("nan")),
    dict(head_dim=64, device="cpu")])
def test_rotaries_that_are_refused(args):
    with pytest.raises(ValueError):
        Rotary(args.pop("head_dim"), **args)


def rotary(**change):
    r = dict(turns=64, axes=None, rotary_dim=64, n_axes=1, pairs=0, scaling=1.0)
    return nat.Rotary(**{**r, **change})


def call(r, x=64, dtype=nat.PP_F16, tokens=3, heads=2, D=64, pos=64, pos_type=nat.PP_POS_I64, out=64):
    return nat.lib().pp_rotate(x, 128, 64, dtype, tokens, heads, D, C.addressof(r) if r else None, pos, 0, pos_type, out,
                               128, 64, None)


@pytest.mark.parametrize("change", [dict(turns=None), dict(turns=68), dict(rotary_dim=24), dict(rotary_dim=0), dict(rotary_dim=80),
                                    dict(n_axes=0), dict(n_axes=2), dict(n_axes=256, axes=64), dict(pairs=2)])
def test_rotary_structs_that_are_refused(change):
    assert call(rotary(**change)) == nat.PP_EINVAL
    assert b"rotary" in nat.lib().pp_last_error()


@pytest.mark.parametrize("change", [dict(x=None), dict(out=None), dict(x=65), dict(out=65), dict(dtype=9), dict(tokens=-1),
                                    dict(tokens=2 ** 28 + 1), dict(heads=-1), dict(heads=65536), dict(D=60), dict(D=520),
                                    dict(D=8), dict(pos=None), dict(pos=68), dict(pos_type=5)])
def test_rows_that_are_refused(change):
    assert call(rotary(), **change) == nat.PP_EINVAL
    assert call(None) == nat.PP_EINVAL


def test_no_rows():
    assert call(rotary(), tokens=0) == nat.PP_OK and call(rotary(), heads=0) == nat.PP_OK


def test_layout_of_the_struct():
    assert [getattr(nat.Rotary, f).offset for f, _ in nat.Rotary._fields_] == [0, 8, 16, 20, 24, 28]
    assert C.sizeof(nat.Rotary) == 32
