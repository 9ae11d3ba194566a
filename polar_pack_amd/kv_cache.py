"""An 8-bit key/value cache and the attention that reads it.

The cache is paged: a page holds ``block`` tokens of every head, one byte a value, with one float32
scale for each page and head of the keys and of the values.  A sequence is a row of a block table;
the packed models of a stream are rows of one table, so that one launch serves all of them.

* :class:`KVCache`       -- the pages
* :func:`kv_append`      -- new keys and values of a step or a prompt
* :func:`kv_attention`   -- attention of the new tokens to everything before and among them
* :func:`kv_read`        -- tokens of the cache as plain values

All three take the same description of a call: ``block_table`` (B, width) int32, ``lengths`` (B,)
int32 (the tokens of each sequence *after* the call's own) and ``cu`` (B + 1,) int32, the offsets of
each sequence's tokens among the call's (None: one token each).  They stay on the device; nothing
here waits for it, and every call can be captured in a HIP graph.  What the three tensors hold is
held to its range on the device: a page outside the cache, or a token past the table, is not
written, reads zero and is attended by no row.

They serve: none has a backward pass, and what they return carries no gradient, whether their
arguments ask for one or not.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _native as nat

BLOCKS = (16, 32, 64, 128)
HEAD_DIMS = (64, 128, 192, 256)
_CODES = {torch.int8: nat.PP_KV_INT8, torch.float8_e4m3fn: nat.PP_KV_E4M3}
_VALUES = {torch.float16: nat.PP_F16, torch.bfloat16: nat.PP_BF16}
_READS = {torch.float16: nat.PP_F16, torch.bfloat16: nat.PP_BF16, torch.float32: nat.PP_F32}


class KVCache:
    """The pages of a cache.

    ``k`` codes (pages, heads, block, D) and ``v`` codes (pages, heads, D, block), int8 or
    float8_e4m3fn; ``k_scale`` and ``v_scale`` float32 (pages, heads).  A value is code * scale.
    Scales are 2**-64 or more (smaller ones count as that in an attention's values) or not finite, and
    the value scales of the pages that one row sees are within a factor of 2**100 (past that its sum of
    weights loses the pages of the smaller ones);
    codes of tokens before a sequence's length are finite, as :func:`kv_append` writes them: a NaN code put
    there by other means may reach rows that do not see it.  What lies past the lengths may hold anything.
    :meth:`zeros` makes a cache; the constructor takes tensors that a program holds already.
    """

    def __init__(self, k, v, k_scale, v_scale):
        if k.dim() != 4 or k.dtype not in _CODES:
            raise TypeError("k must be int8 or float8_e4m3fn (pages, heads, block, D)")
        pages, heads, block, D = k.shape
        if block not in BLOCKS or D not in HEAD_DIMS:
            raise ValueError(f"block must be one of {BLOCKS} and D one of {HEAD_DIMS}, got {block} and {D}")
        if v.dtype != k.dtype or v.shape != (pages, heads, D, block):
            raise ValueError("v must have k's type and the shape (pages, heads, D, block)")
        for s in (k_scale, v_scale):
            if s.dtype != torch.float32 or s.shape != (pages, heads):
                raise ValueError("scales must be float32 (pages, heads)")
        ts = (k, v, k_scale, v_scale)
        if k.device.type != "cuda" or any(t.device != k.device for t in ts):
            raise ValueError("a cache's tensors must be on one ROCm device")
        if not all(t.is_contiguous() and not t.is_neg() for t in ts):
            raise ValueError("a cache's tensors must be contiguous and hold their values as they are")
        if pages < 1 or heads < 1 or k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("a cache needs a page and a head, and codes at 16-byte boundaries")
        self.k, self.v, self.k_scale, self.v_scale = ts
        self.pages, self.heads, self.block, self.head_dim = pages, heads, block, D
        self.device = k.device
        self._abi = nat.KVCache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, heads, D,
                                block, _CODES[k.dtype])
        self._ref = ctypes.addressof(self._abi)

    @classmethod
    def zeros(cls, pages, heads, head_dim, *, block=64, dtype=torch.int8, device="cuda"):
        k = torch.zeros(pages, heads, block, head_dim, dtype=torch.int8, device=device)
        v = torch.zeros(pages, heads, head_dim, block, dtype=torch.int8, device=device)
        k_scale, v_scale = (torch.zeros(pages, heads, dtype=torch.float32, device=device) for _ in range(2))
        return cls(k.view(dtype), v.view(dtype), k_scale, v_scale)


def _check_cache(cache):
    if not isinstance(cache, KVCache):
        raise TypeError("cache must be a KVCache")


def _call(cache, block_table, lengths, cu, tokens):
    """The checked description of a call: (table, row stride, width, lengths, cu, B) for the C entries."""
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise TypeError("block_table must be int32 (B, width) and lengths int32 (B,)")
    B, width = block_table.shape
    dev = cache.device
    if lengths.shape != (B,) or lengths.stride(0) != 1 and B > 1 or block_table.stride(1) != 1 and width > 1:
        raise ValueError("lengths must be a contiguous (B,) tensor and block_table's rows contiguous")
    if block_table.device != dev or lengths.device != dev:
        raise ValueError("all operands must be on the cache's device")
    if B < 1 or width < 1:
        raise ValueError("block_table must hold a sequence and a page")
    if cu is None:
        if tokens != B:
            raise ValueError(f"{tokens} tokens for {B} sequences: cu must say which are whose")
        return block_table.data_ptr(), block_table.stride(0), width, lengths.data_ptr(), None, B
    if cu.dtype != torch.int32 or cu.shape != (B + 1,) or not cu.is_contiguous():
        raise TypeError("cu must be a contiguous int32 (B + 1,) tensor")
    if cu.device != dev:
        raise ValueError("all operands must be on the cache's device")
    return block_table.data_ptr(), block_table.stride(0), width, lengths.data_ptr(), cu.data_ptr(), B


def _values(cache, x, name, heads):
    """A (tokens, heads, D) tensor of 16-bit values with a contiguous last dimension."""
    if x.dim() != 3 or x.dtype not in _VALUES:
        raise TypeError(f"{name} must be float16 or bfloat16 (tokens, heads, D)")
    if x.shape[2] != cache.head_dim or heads is not None and x.shape[1] != heads:
        raise ValueError(f"{name} must be (tokens, {heads if heads else 'heads'}, {cache.head_dim})")
    if x.device != cache.device:
        raise ValueError("all operands must be on the cache's device")
    if x.is_neg():                                   # memory that holds the values negated
        x = x.resolve_neg()
    return x if x.stride(2) == 1 else x.contiguous()


def kv_append(cache, k, v, block_table, lengths, cu=None):
    """Write the call's keys and values (tokens, heads, D), float16 or bfloat16, into the cache.

    For each page and head that gets tokens, k and v apart, in float32::

        scale = max(old scale, max|x| / qmax, 2**-64)      qmax 127 (int8) or 448 (e4m3)
        code  = round(x * f)                               ties to even, held to +-qmax

    with f = qmax / max|x| where that sets the scale and 1 / scale otherwise.  The old scale counts
    where the page holds earlier tokens of the sequence; where it grows their codes become
    ``round(code * (old / scale))``.  A value that is not finite makes its page's scale
    not finite, so that every row that sees the page is NaN.  A page that gets tokens must belong
    to one sequence of the call (shared pages are for tokens already written).
    """
    _check_cache(cache)
    k = _values(cache, k, "k", cache.heads)
    v = _values(cache, v, "v", cache.heads)
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError("k and v must have one shape and type")
    n = k.shape[0]
    call = _call(cache, block_table, lengths, cu, n)
    with nat.on_device(cache.device):
        nat.check(nat.lib().pp_kv_append(cache._ref, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                                         v.stride(0), v.stride(1), _VALUES[k.dtype], n, *call,
                                         nat.raw_stream(cache.device)), "pp_kv_append")


def kv_read(cache, block_table, lengths, cu=None, *, total=None, dtype=torch.float16):
    """(k, v), each (total, heads, D): the values of the last ``cu[b + 1] - cu[b]`` tokens of each
    sequence, code * scale rounded once to ``dtype``.  ``total`` is ``cu[B]``, a number that the
    program holds (the call does not wait for the device to learn it)."""
    _check_cache(cache)
    if dtype not in _READS:
        raise TypeError("dtype must be float16, bfloat16 or float32")
    if total is None:
        if cu is not None:
            raise ValueError("total must be given with cu")
        total = block_table.shape[0]
    call = _call(cache, block_table, lengths, cu, total)
    with nat.on_device(cache.device):
        out = torch.empty((2, total, cache.heads, cache.head_dim), dtype=dtype, device=cache.device)
        k, v = out.unbind(0)
        nat.check(nat.lib().pp_kv_read(cache._ref, *call, total, _READS[dtype], k.data_ptr(), v.data_ptr(),
                                       nat.raw_stream(cache.device)), "pp_kv_read")
    return k, v


def kv_attention(q, cache, block_table, lengths, cu=None, *, causal=True, window=0, scale=None, return_lse=False):
    """Attention of the call's queries ``q`` (tokens, q_heads, D), float16 or bfloat16, to the cache.

    Query head ``hq`` reads head ``hq // (q_heads // heads)``.  The call's i-th token of sequence b has
    position ``p = lengths[b] - n_b + i`` and sees the keys of ``[0, p]``, with ``window > 0`` only the
    last ``window`` of them, with ``causal=False`` all ``lengths[b]``.  Causal or not, the call's tokens are
    the last ones of their sequence: one whose position is negative, where a sequence has more queries than
    ``lengths[b]``, is no token of it and sees nothing (as it is not written and reads zero).  Queries that are
    not the sequence's own, as in attention to another text, are passed at most ``lengths[b]`` a call.
    ``scale`` defaults to ``D ** -0.5``.  A row that sees no key is zero (lse -inf).

    Returns (tokens, q_heads, D) of q's type, and with ``return_lse`` also the float32 (tokens,
    q_heads) natural logarithms of the sums, by which attention over several caches is joined.
    """
    _check_cache(cache)
    q = _values(cache, q, "q", None)
    n, heads = q.shape[0], q.shape[1]
    if heads == 0 or heads % cache.heads:
        raise ValueError(f"{heads} query heads over {cache.heads} heads")
    if window < 0 or window and not causal:
        raise ValueError("window must be 0 or a positive length of causal attention")
    call = _call(cache, block_table, lengths, cu, n)
    scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale)
    dev = cache.device
    with nat.on_device(dev):
        out = torch.empty((n, heads, cache.head_dim), dtype=q.dtype, device=dev)
        lse = torch.empty((n, heads), dtype=torch.float32, device=dev) if return_lse else None
        shape = (dev.index, cache.heads, cache.head_dim, cache.block, call[2], call[5], n, heads)
        size = nat.sized("pp_kv_attention_workspace_size", *shape)
        n_counts = nat.sized("pp_kv_attention_counts_size", *shape)
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        counts, key = nat.zero_workspace(dev, n_counts)
        rc = nat.lib().pp_kv_attention(cache._ref, q.data_ptr(), q.stride(0), q.stride(1), heads, _VALUES[q.dtype], n,
                                       *call, int(causal), int(window), scale, out.data_ptr(),
                                       lse.data_ptr() if return_lse else None, ws.data_ptr() if size else None, size,
                                       counts.data_ptr() if n_counts else None, n_counts, nat.raw_stream(dev))
        if rc:
            nat.drop_workspace(key)
        nat.check(rc, "pp_kv_attention")
    return (out, lse) if return_lse else out
