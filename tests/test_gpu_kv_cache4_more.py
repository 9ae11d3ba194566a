"""The 4-bit cache where the first tests of it do not look: turned keys that lie next to a border between two codes, and
drafts that are written over."""
import math
from fractions import Fraction

import pytest
import torch

from polar_pack_amd.kv_cache import KVCache4, kv_read, kv_rotate_append
from polar_pack_amd.rotary import Rotary
from serving import DEV
from serving4 import unpack

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


def test_drafts_that_were_refused_leave_nothing():
    """Steps append five drafted tokens, of which some stay and the next step writes over the rest, not finite ones among
    them: what lies below the length is byte for byte what one append of the tokens that stayed leaves."""
    H, D, bs, n = 2, 64, 16, 60
    g = torch.Generator().manual_seed(9)
    k, v, q = (torch.randn(n, h, D, generator=g).half().to(DEV) for h in (H, H, 3))
    r, table = Rotary(D), torch.tensor([[2, 0, 4, 1, 3]], dtype=torch.int32, device=DEV)
    lengths = lambda m: torch.tensor([m], dtype=torch.int32, device=DEV)
    cu = lambda m: torch.tensor([0, m], dtype=torch.int32, device=DEV)
    whole, steps = (KVCache4.zeros(5, H, D, block=bs, device=DEV) for _ in range(2))
    want = kv_rotate_append(whole, q, k, v, r, table, lengths(n), cu(n))
    at, i, turned = 0, 0, []
    while at < n:
        stay = min([3, 1, 5, 2, 4][i % 5], n - at)
        kk, vv, qq = (torch.randn(5, h, D, generator=g).half().to(DEV) * 5 for h in (H, H, 3))
        kk[:stay], vv[:stay], qq[:stay] = k[at:at + stay], v[at:at + stay], q[at:at + stay]
        if stay < 5:
            (kk if i % 2 else vv)[4, i % H, 7] = float("nan" if i % 3 else "inf")
        turned.append(kv_rotate_append(steps, qq, kk, vv, r, table, lengths(at + 5), cu(5))[:stay])
        at, i = at + stay, i + 1
    assert torch.equal(torch.cat(turned), want)
    for p in range(5):
        page, seen = int(table[0, p]), min(max(n - p * bs, 0), bs)
        for name, axis in (("k", 1), ("k_scale", 1), ("v_scale", 2)):
            a, b = (getattr(c, name).view(torch.uint8)[page].narrow(axis, 0, seen) for c in (steps, whole))
            assert torch.equal(a, b), (p, name)
        a, b = (unpack(c.v[page].cpu())[..., :seen] for c in (steps, whole))
        assert torch.equal(a, b), p
