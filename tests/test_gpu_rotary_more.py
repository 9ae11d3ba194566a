"""rotate where the first tests of it do not look: how frequencies are given, the farthest positions, tensors that a
backward pass has saved."""
from fractions import Fraction

import numpy as np
import pytest
import torch

from polar_pack_amd.rotary import Rotary, _turn, rotate
from serving import DEV
from serving4 import PI, partners

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("place", ["x", "other"])
def test_a_saved_tensor_that_is_written_over_is_noticed(place):
    leaf = torch.randn(3, 2, 64, device=DEV, requires_grad=True)
    saved = leaf * 2.0
    loss = (saved * saved).sum()                              # keeps `saved` for its gradient
    x, r, pos = (saved if place == "x" else torch.randn(3, 2, 64, device=DEV)), Rotary(64), torch.arange(3, device=DEV)
    want = rotate(x.detach().clone(), r, pos)
    assert torch.equal(rotate(x, r, pos, out=saved), want)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_tensors_without_versions():
    """Made in inference mode they have none, in or outside of it."""
    r, pos = Rotary(64), torch.arange(3, device=DEV)
    with torch.inference_mode():
        x = torch.randn(3, 2, 64, device=DEV)
        want = rotate(x, r, pos)
        assert torch.equal(rotate(x, r, pos, out=torch.empty_like(x)), want)
    other = torch.empty(3, 2, 64, device=DEV)
    assert torch.equal(rotate(x, r, pos, out=other), want)
    assert torch.equal(rotate(x, r, pos, out=x), want)


@pytest.mark.parametrize("kind", [list, tuple, np.array, lambda f: [torch.tensor(x, dtype=torch.float64) for x in f]])
def test_frequencies_keep_their_bits(kind):
    """Numbers of 64 bits, however they are given: the default ones, given, turn far positions as the default ones do."""
    freqs = [10000.0 ** (-f / 32) for f in range(32)]
    x, pos = torch.randn(4, 2, 64, device=DEV), torch.tensor([1, 4097, 10 ** 6 + 1, -2 ** 40], device=DEV)
    want = rotate(x, Rotary(64), pos)
    assert torch.equal(rotate(x, Rotary(64, inv_freq=kind(freqs)), pos), want)
    assert torch.equal(rotate(x, Rotary(64, inv_freq=torch.tensor(freqs, dtype=torch.float64)), pos), want)


def test_frequencies_of_32_bits_are_what_they_are():
    freqs = torch.tensor([10000.0 ** (-f / 32) for f in range(32)])
    x, pos = torch.randn(2, 2, 64, device=DEV), torch.tensor([4097, 10 ** 6 + 1], device=DEV)
    want = rotate(x, Rotary(64, inv_freq=freqs.double()), pos)
    assert torch.equal(rotate(x, Rotary(64, inv_freq=freqs), pos), want)
    assert torch.equal(rotate(x, Rotary(64, inv_freq=freqs.numpy()), pos), want)


@pytest.mark.parametrize("pos", [2 ** 62, 2 ** 63 - 1, -2 ** 63, 2 ** 55 + 3, -2 ** 47 - 1])
def test_the_farthest_positions(pos):
    """Of the fraction of a turn that is held, the angle keeps all its bits at any position: sines and cosines are off by no
    more than near zero (the bound of the other tests; a 64-bit angle and its sine in the reference add 2^-51)."""
    x = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(6))
    freqs = [10000.0 ** (-f / 32) for f in range(32)]
    rest = [Fraction(_turn(f) * pos % 2 ** 64, 2 ** 64) for f in freqs]
    a = torch.tensor([float((t - 1 if 2 * t > 1 else t) * 2 * PI) for t in rest], dtype=torch.float64)
    c, s, v = torch.cos(a), torch.sin(a), x.double()
    want = torch.cat([v[..., :32] * c - v[..., 32:] * s, v[..., 32:] * c + v[..., :32] * s], 2)
    got = rotate(x.to(DEV), Rotary(64), torch.tensor([pos], device=DEV)).cpu().double()
    assert ((got - want).abs() <= (2.0 ** -22 + 2.0 ** -50) * partners(v, 64, "halves") + 2.0 ** -24 * want.abs()).all()
