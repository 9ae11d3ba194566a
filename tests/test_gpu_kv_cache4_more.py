"""The 4-bit cache where the first tests of it do not look: turned keys that lie next to a border between two codes."""
import math
from fractions import Fraction

import pytest
import torch

from polar_pack_amd.kv_cache import KVCache4, kv_read, kv_rotate_append
from polar_pack_amd.rotary import Rotary
from serving import DEV

pytestmark = pytest.mark.gpu


def cosine(x):
    """Of a small rational number, to 2^-100."""
    total, term, n = Fraction(0), Fraction(1), 0
    while abs(term) > Fraction(1, 2 ** 110):
        total += term
        term = -term * x * x / ((n + 1) * (n + 2))
        n += 2
    return total


def beside(border):
    """(key, angle): keys whose first value, key * cos(angle) near an eighth of a turn, lies above `border` by 5 to 7 parts in
    10^16.  A cosine within 1.9e-16, times the key and rounded to 64 bits, is off by less than 1.42 * 1.9e-16 + 1.2e-16 of the
    border, so the value is on the border's upper side."""
    found = []
    key = math.ceil(border * 1.4001 * 256) / 256
    while key < border * 1.4140 and len(found) < 3:
        angle = math.acos(border / key)
        while cosine(Fraction(angle)) * Fraction(key) < Fraction(border) * (1 + Fraction(5, 10 ** 16)):
            angle = math.nextafter(angle, 0)
        while cosine(Fraction(angle)) * Fraction(key) > Fraction(border) * (1 + Fraction(7, 10 ** 16)):
            angle = math.nextafter(angle, 1)
        above = cosine(Fraction(angle)) * Fraction(key) / Fraction(border) - 1
        if Fraction(5, 10 ** 16) <= above <= Fraction(7, 10 ** 16) and angle > 0.775 and torch.tensor(key).half().item() == key:
            found.append((key, angle))
        key += 1 / 256
    return found


def test_turned_keys_beside_a_border():
    """Codes are the nearest to the keys in 64 bits, so the cosines must have all of those near an eighth of a turn too."""
    borders = {0.75: 1.0, 1.25: 1.5, 1.75: 2.0, 2.5: 3.0, 3.5: 4.0}
    cases = [(key, angle, up) for border, up in borders.items() for key, angle in beside(border)]
    assert len(cases) >= 10
    cases = cases[:31]
    k = torch.zeros(1, 1, 64, dtype=torch.float16)
    k[0, 0, 31] = 6.0                                             # sets the scale, 1
    freqs = [angle for _, angle, _ in cases] + [0.0] * (32 - len(cases))
    for f, (key, _, _) in enumerate(cases):
        k[0, 0, f] = key
    cache, r = KVCache4.zeros(1, 1, 64, block=16, device=DEV), Rotary(64, inv_freq=torch.tensor(freqs, dtype=torch.float64))
    at = (torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV))
    kv_rotate_append(cache, None, k.to(DEV), torch.zeros_like(k).to(DEV), r, *at,
                     positions=torch.ones(1, dtype=torch.int64, device=DEV))
    got = kv_read(cache, *at, dtype=torch.float32)[0][0, 0].tolist()
    assert got[31] == 6.0
    assert got[:len(cases)] == [up for _, _, up in cases]
