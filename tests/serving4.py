"""Plain forms of rotary positions and of the 4-bit cache for their tests: 64-bit, on the CPU, written from the
definitions."""
import math
from fractions import Fraction

import torch

from serving import DEV

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _pi(bits):
    """pi * 2^bits by Machin's formula in whole numbers."""
    one = 1 << (bits + 20)

    def arctan(n):
        term, total, k = one // n, one // n, 1
        while term:
            term = -term // (n * n)
            k += 2
            total += term // k
        return total
    return 4 * (4 * arctan(5) - arctan(239)) >> 20


PI = Fraction(_pi(160), 1 << 160)


def angles(freqs, positions):
    """(tokens, freqs) angles in (-pi, pi] for whole positions of any size, one rounding each."""
    rows = []
    for ps in positions:
        row = []
        for f, p in zip(freqs, ps):
            turns = Fraction(f) * p / (2 * PI) % 1
            row.append(float((turns - 1 if turns > Fraction(1, 2) else turns) * 2 * PI))
        rows.append(row)
    return torch.tensor(rows, dtype=torch.float64)


def turn(x, rot, pairs, freqs, axes, positions, scaling=1.0):
    """x (tokens, heads, D) float64 turned; positions: a list of whole numbers for each axis."""
    a = angles(freqs, [[positions[ax][t] for ax in axes] for t in range(x.shape[0])])
    c, s = (torch.cos(a) * scaling)[:, None], (torch.sin(a) * scaling)[:, None]
    out = x.clone()
    lo, hi = ((slice(0, rot // 2), slice(rot // 2, rot)) if pairs == "halves" else (slice(0, rot, 2), slice(1, rot, 2)))
    out[..., lo] = x[..., lo] * c - x[..., hi] * s
    out[..., hi] = x[..., hi] * c + x[..., lo] * s
    return out


def partners(x, rot, pairs):
    """|a| + |b| of the pair that each value belongs to (what is not turned: 0)."""
    out = torch.zeros_like(x)
    lo, hi = ((slice(0, rot // 2), slice(rot // 2, rot)) if pairs == "halves" else (slice(0, rot, 2), slice(1, rot, 2)))
    out[..., lo] = out[..., hi] = x[..., lo].abs() + x[..., hi].abs()
    return out


def code4(x):
    """(codes 0..15, scales) of rows (..., D) float64, a group of 32 and a value at a time by the definition."""
    v = x.unflatten(-1, (-1, 32))
    top = v.abs().amax(-1)
    scale = torch.full_like(top, 2.0 ** 13)
    for e in range(12, -15, -1):
        scale = torch.where(top <= 7 * 2.0 ** e, 2.0 ** e, scale)
    t = (v / scale[..., None]).abs().clamp(max=6.0)
    dist = (t[..., None] - E2M1).abs()
    best = dist.amin(-1, keepdim=True)
    near = dist == best                                       # two where it is halfway: the even code
    even = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])             # codes, the even ones first
    code = even[near[..., even].int().argmax(-1)]
    return (code + 8 * (torch.signbit(v)).int()).flatten(-2), scale


def value4(codes):
    return E2M1[(codes & 7).long()] * torch.where(codes >= 8, -1.0, 1.0)


def unpack(b):
    """Bytes (..., n) to codes (..., 2 n), the low half first."""
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def pack(codes):
    c = codes.to(torch.uint8)
    return c[..., 0::2] | c[..., 1::2] << 4


def random_cache4(pages, H, bs, D, g, low=-3, high=1):
    """Host tensors (k, v, k_scale, v_scale)."""
    k = torch.randint(0, 256, (pages, H, bs, D // 2), generator=g, dtype=torch.uint8)
    v = torch.randint(0, 256, (pages, H, D, bs // 2), generator=g, dtype=torch.uint8)
    ks, vs = (torch.exp2(torch.randint(low, high, s, generator=g).float()).to(torch.float8_e5m2)
              for s in ((pages, H, bs, D // 32), (pages, H, D // 32, bs)))
    return k, v, ks, vs


def device_cache4(parts):
    from polar_pack_amd.kv_cache import KVCache4
    return KVCache4(*[t.to(DEV) for t in parts])


def f8(t):
    """float8 as float64 (indexing it is done on its bytes)."""
    return t.view(torch.uint8).view(torch.float8_e5m2).double()


def plain_parts(parts):
    """The cache as one of plain values and scales of 1, for the plain forms of the 8-bit cache: values of tokens
    that are marked are NaN."""
    k, v, ks, vs = parts
    K = value4(unpack(k)) * f8(ks).repeat_interleave(32, -1)
    V = value4(unpack(v)) * f8(vs).repeat_interleave(32, 2)
    marked = f8(ks).isnan().any(-1)
    K[marked] = 0.0
    V = torch.where(marked[:, :, None, :], math.nan, V)
    one = torch.ones(k.shape[:2])
    return K, V, one, one


def append4(parts, k, v, table, lens, news):
    """The cache after an append of float64 keys and values (tokens, heads, D)."""
    out = [t.clone() for t in parts]
    pages, H, bs = parts[0].shape[:3]
    kb, vb, ks, vs = out[0], out[1], out[2].view(torch.uint8), out[3].view(torch.uint8)
    at = 0
    for b, n in enumerate(news):
        for i in range(n):
            pos = lens[b] - n + i
            p = int(table[b, pos // bs]) if 0 <= pos < table.shape[1] * bs else -1
            if not 0 <= p < pages:
                continue
            t = pos % bs
            bad = ~(k[at + i].isfinite().all(-1) & v[at + i].isfinite().all(-1))       # (H,)
            ck, sk = code4(k[at + i].nan_to_num(0, 0, 0))
            cv, sv = code4(v[at + i].nan_to_num(0, 0, 0))
            byte = sk.to(torch.float8_e5m2).view(torch.uint8)
            ks[p, :, t] = torch.where(bad[:, None], 127, byte)
            keep = ~bad                                       # what a token that is not finite leaves as codes is open
            kb[p, keep, t] = pack(ck)[keep]
            old = vb[p, :, :, t // 2]
            new = (old & 15 | cv << 4) if t % 2 else (old & 240 | cv)
            vb[p, keep, :, t // 2] = new.to(torch.uint8)[keep]
            vs[p, keep, :, t] = sv.to(torch.float8_e5m2).view(torch.uint8)[keep]
        at += n
    return out
