"""Rotary positions, of one axis or several (time, height and width of images and video).

* :class:`Rotary`  -- which values turn with which frequency and axis
* :func:`rotate`   -- rows of queries or keys turned by their positions

:func:`polar_pack_amd.kv_cache.kv_rotate_append` does the same on the way into a cache.  They serve:
none has a backward pass, and what they return carries no gradient.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _native as nat

HEAD_DIM_MAX = 512
_ROWS = {torch.float16: nat.PP_F16, torch.bfloat16: nat.PP_BF16, torch.float32: nat.PP_F32}
_POSITIONS = {torch.int32: nat.PP_POS_I32, torch.int64: nat.PP_POS_I64}
_PAIRS = {"halves": nat.PP_PAIRS_HALVES, "neighbours": nat.PP_PAIRS_NEIGHBOURS}
# 2^124 / (2 pi), cut off: a larger frequency's fraction of a turn would be off by more than its rounding to 2^-65
_TURN = 0x28BE60DB9391054A7F09D5F47D4D377
_FREQ_MAX = 2.0 ** 58


def _turn(freq):
    """The fraction of a turn that ``freq`` radians are, times 2^64 and rounded, as a signed 64-bit number."""
    n, d = freq.as_integer_ratio()                   # d is a power of two
    shift = 60 + d.bit_length() - 1
    t = ((n * _TURN + (1 << (shift - 1))) >> shift) & ((1 << 64) - 1)
    return t - (1 << 64) if t >= 1 << 63 else t


class Rotary:
    """How rows of ``head_dim`` values turn.

    The first ``rotary_dim`` values (a multiple of 16; default all) are turned in pairs, value f with
    ``f + rotary_dim / 2`` (``pairs="halves"``) or 2f with 2f + 1 (``"neighbours"``), pair f by
    ``position * inv_freq[f]`` radians::

        a' = scaling * (a cos - b sin)        b' = scaling * (b cos + a sin)

    with ``scaling`` held in float32.  ``inv_freq`` holds rotary_dim / 2 numbers up to 2**58, by default
    ``base ** (-2 f / rotary_dim)``; other spacings (stretched contexts) are given that way.  With several axes a
    token has a position on each: ``sections`` says how many frequencies each axis turns, one axis after
    another, or ``axes`` names the axis of every frequency (in turn, say).

    There is no table of positions, and any 64-bit position is taken.  A frequency is held to 2**-65 of a turn, so the
    angle of a position is off by up to ``abs(position) * 2**-65`` turns, 2e-13 radians at 10**6.  Below 2**38
    that is less than a sine in float32 is off by; at 2**62 it is most of a radian.
    """

    def __init__(self, head_dim, *, base=10000.0, rotary_dim=None, inv_freq=None, sections=None, axes=None,
                 pairs="halves", scaling=1.0, device="cuda"):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if not 16 <= head_dim <= HEAD_DIM_MAX or head_dim % 8:
            raise ValueError(f"head_dim must be a multiple of 8 in 16..{HEAD_DIM_MAX}, got {head_dim}")
        if not 16 <= rotary_dim <= head_dim or rotary_dim % 16:
            raise ValueError(f"rotary_dim must be a multiple of 16 up to head_dim, got {rotary_dim}")
        if pairs not in _PAIRS:
            raise ValueError("pairs must be 'halves' or 'neighbours'")
        n = rotary_dim // 2
        if inv_freq is None:
            if not (math.isfinite(base) and base > 0):
                raise ValueError("base must be a positive number")
            freq = [float(base) ** (-f / n) for f in range(n)]
        else:
            if not torch.is_tensor(inv_freq):        # Python's numbers would become float32
                inv_freq = torch.as_tensor(inv_freq, dtype=torch.float64)
            freq = [float(f) for f in inv_freq.detach().double().cpu().reshape(-1)]
        if len(freq) != n or not all(abs(f) <= _FREQ_MAX for f in freq):
            raise ValueError(f"inv_freq must hold {n} numbers within +-2**58")
        if sections is not None and axes is not None:
            raise ValueError("give sections or axes, not both")
        if sections is not None:
            sections = [int(s) for s in sections]
            if any(s < 0 for s in sections) or sum(sections) != n:
                raise ValueError(f"sections must add up to {n} frequencies")
            axes = [a for a, s in enumerate(sections) for _ in range(s)]
            self.n_axes = len(sections)
        else:
            axes = [0] * n if axes is None else [int(a) for a in axes]
            self.n_axes = max(axes, default=0) + 1
        if len(axes) != n or not 1 <= self.n_axes <= 255 or min(axes) < 0:
            raise ValueError(f"axes must hold {n} numbers from 0 to 254")
        if not abs(scaling) <= torch.finfo(torch.float32).max:
            raise ValueError("scaling must be a float32 number")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("a Rotary lives on a ROCm device (device.type == 'cuda')")
        self.head_dim, self.rotary_dim, self.pairs, self.scaling = head_dim, rotary_dim, pairs, float(scaling)
        turns = torch.tensor([_turn(f) for f in freq], dtype=torch.int64)
        self._turns = turns.to(device)
        self._axes = None if self.n_axes == 1 else torch.tensor(axes, dtype=torch.uint8).to(device)
        self.device = self._turns.device
        self._abi = nat.Rotary(self._turns.data_ptr(), self._axes.data_ptr() if self._axes is not None else None,
                               rotary_dim, self.n_axes, _PAIRS[pairs], self.scaling)
        self._ref = ctypes.addressof(self._abi)


def _check_rotary(rotary, head_dim, device):
    if not isinstance(rotary, Rotary):
        raise TypeError("rotary must be a Rotary")
    if rotary.head_dim != head_dim:
        raise ValueError(f"rotary is of head_dim {rotary.head_dim}, the rows are of {head_dim}")
    if rotary.device != device:
        raise ValueError("all operands must be on one ROCm device")


def _positions(rotary, positions, tokens, device):
    """(address, stride between axes, type) of (tokens,) or (axes, tokens) positions, and the tensor that holds them."""
    if positions.dtype not in _POSITIONS:
        raise TypeError("positions must be int32 or int64")
    one = rotary.n_axes == 1 and positions.dim() == 1
    if positions.shape != ((tokens,) if one else (rotary.n_axes, tokens)):
        raise ValueError(f"positions must be ({rotary.n_axes}, {tokens})" + (f" or ({tokens},)" if rotary.n_axes == 1 else ""))
    if positions.device != device:
        raise ValueError("all operands must be on one ROCm device")
    if positions.stride(-1) != 1 and tokens > 1:
        positions = positions.contiguous()
    return positions, (positions.data_ptr(), 0 if one else positions.stride(0), _POSITIONS[positions.dtype])


def rotate(x, rotary, positions, *, out=None):
    """Rows ``x`` (tokens, heads, head_dim), float16, bfloat16 or float32, turned by ``positions``.

    ``positions`` int32 or int64: (tokens,) with one axis, (axes, tokens) with several; any numbers, negative ones
    turn back.  Computed in float32, sines and cosines within 1e-7, and rounded once to x's type.  ``out`` takes
    the result: x itself, or a tensor of its shape and type in a storage of its own (another slice of the tensor
    that x is a slice of is refused); by default a new one.  A backward pass that has saved ``out`` raises then, as
    after torch's own writes in place.
    """
    if x.dim() != 3 or x.dtype not in _ROWS:
        raise TypeError("x must be float16, bfloat16 or float32 (tokens, heads, head_dim)")
    dev = x.device
    if dev.type != "cuda":
        raise ValueError("x must be on a ROCm device (tensor.device.type == 'cuda')")
    tokens, heads, D = x.shape
    _check_rotary(rotary, D, dev)
    positions, at = _positions(rotary, positions, tokens, dev)
    given = out is not None
    if given:
        if out.shape != x.shape or out.dtype != x.dtype or out.device != dev:
            raise ValueError("out must have x's shape, type and device")
        if out.stride(2) != 1 or out.is_neg():
            raise ValueError("out must hold its values as they are, a row's one after another")
        same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride() and not x.is_neg()
        if not same and out.untyped_storage().data_ptr() == x.untyped_storage().data_ptr():
            raise ValueError("out must be x itself or lie in another storage than x's")
        reach = D                                    # of the rows along the nearer stride, then along both
        for step, rows in sorted((out.stride(i), out.shape[i]) for i in (0, 1) if out.numel() and out.shape[i] > 1):
            if step < reach:
                raise ValueError("out's rows must not overlap")
            reach += step * (rows - 1)
    if x.is_neg():                                   # memory that holds the values negated
        x = x.resolve_neg()
    st, sh, sd = x.stride()
    if sd != 1:
        x = x.contiguous()
        st, sh, _ = x.stride()
    with nat.on_device(dev):
        if out is None:
            out, o_st, o_sh = torch.empty_like(x, memory_format=torch.contiguous_format), heads * D, D
        else:
            o_st, o_sh, _ = out.stride()
        nat.check(nat.lib().pp_rotate(x.data_ptr(), st, sh, _ROWS[x.dtype], tokens, heads, D, rotary._ref, *at,
                                      out.data_ptr(), o_st, o_sh, nat.raw_stream(dev)), "pp_rotate")
    if given and not out.is_inference():             # a backward pass that has saved it says so instead of using it
        torch.autograd.graph.increment_version(out)
    return out
