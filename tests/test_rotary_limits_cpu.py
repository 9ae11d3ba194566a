"""Numbers that a Rotary cannot hold are refused before any device is asked; those it can are held to their last bit."""
import ctypes as C
from fractions import Fraction

import pytest

from polar_pack_amd import _native as nat
from polar_pack_amd.rotary import Rotary, _turn
from serving4 import _pi


@pytest.mark.parametrize("args", [dict(scaling=1e39), dict(scaling=-3.5e38), dict(scaling=float("inf")), dict(inv_freq=[1e18] * 32),
                                  dict(inv_freq=[-2.0 ** 59] + [0.0] * 31), dict(inv_freq=[float("inf")] * 32), dict(base=1e-300)])
def test_numbers_out_of_range(args):
    """A device that is none is refused last: these are refused for themselves."""
    with pytest.raises(ValueError, match="scaling|inv_freq"):
        Rotary(64, device="cpu", **args)


@pytest.mark.parametrize("args", [dict(scaling=3.4e38), dict(scaling=-1.0), dict(inv_freq=[2.0 ** 58, -2.0 ** 58] * 16)])
def test_numbers_in_range(args):
    with pytest.raises(ValueError, match="ROCm device"):
        Rotary(64, device="cpu", **args)


@pytest.mark.parametrize("freq", [2.0 ** 58, -2.0 ** 58 * (1 - 2.0 ** -53), 1.0, -1.0, 0.1, 1e-5, 6.283185307179586, 2.0 ** -70, 12345.678, 1e17])
def test_fractions_of_a_turn(freq):
    """To the nearest 2^-64 of a turn, 2^-124 * 2^58 of a turn beside it."""
    turns = Fraction(freq) * (1 << 250) / (2 * _pi(250)) * (1 << 64)
    off = (turns - _turn(freq)) % (1 << 64)
    assert min(off, (1 << 64) - off) <= Fraction(1, 2) + Fraction(1, 4)


def test_the_struct_is_as_long_as_the_library_has_it():
    out = (C.c_int64 * 6)()
    assert nat.lib().pp_abi_sizes(out, 6) == 6
    assert out[5] == C.sizeof(nat.Rotary) and out[4] == C.sizeof(nat.KVCache)
