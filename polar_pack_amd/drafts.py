"""Drafted tokens: which of them the target keeps, and the token after them."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as nat

_PROBABILITIES = {torch.float16: nat.PP_F16, torch.bfloat16: nat.PP_BF16, torch.float32: nat.PP_F32}


class Verified(NamedTuple):
    """int64 ``tokens`` (B, n + 1): the accepted drafts, the token after them, then -1; int64 ``accepted`` (B,)."""
    tokens: torch.Tensor
    accepted: torch.Tensor


def _rows(x):
    """A (B, rows, V) tensor whose rows lie one value after another and hold them as they are, and its strides."""
    if x.is_neg():                                   # memory that holds the values negated
        x = x.resolve_neg()
    sb, sr, sv = x.stride()
    if sv != 1 and x.shape[2] > 1:
        x = x.contiguous()
        sb, sr, _ = x.stride()
    return x, sb, sr


def verify_drafts(target, draft, tokens, uniforms, counts=None):
    """Check drafted ``tokens`` (B, n) int64 against the target's probabilities, with given random numbers.

    ``target`` (B, n + 1, V): the target's probabilities at each draft and after the last one; ``draft`` (B, n, V), of
    one type with it (float16, bfloat16 or float32): what the tokens were drawn from, or None where they were certain (an
    argmax, a phrase looked up).  ``uniforms`` float32 (B, n + 1), in [0, 1).  ``counts`` int32 (B,): how many drafts a
    sequence has where that is not n; what lies past them is not read.

    Draft i is kept while ``u_i q_i(token) < p_i(token)``.  The token after the kept ones is drawn with ``u_n``: at a
    refused draft from ``max(p_i - q_i, 0)`` (``draft=None``: from p_i without the token; from p_i where nothing is left),
    after the last from ``p_count``; it is the first whose sum of entries up to it passes ``u_n`` times the sum of all.  So
    the answer is distributed as the target's own.  Sums are held in float64; rows need not add up to one.  A NaN or an
    entry below 0 counts as 0, infinity as the largest float32, a token outside [0, V) has probability 0; from a row of
    nothing the token is -1.  With n = 0 it draws a token from each row.

    Nothing waits for the device, and a call can be captured in a HIP graph.  There is no backward pass.
    """
    if target.dim() != 3 or target.dtype not in _PROBABILITIES:
        raise TypeError("target must be float16, bfloat16 or float32 (B, n + 1, V)")
    B, n, V = target.shape
    n -= 1
    if n < 0 or V < 1:
        raise ValueError("target must have a row for the token after the drafts, and a probability in it")
    if draft is not None and (draft.dtype != target.dtype or draft.shape != (B, n, V)):
        raise ValueError(f"draft must be of target's type and ({B}, {n}, {V})")
    if tokens.dtype != torch.int64 or tokens.shape != (B, n):
        raise TypeError(f"tokens must be int64 ({B}, {n})")
    if uniforms.dtype != torch.float32 or uniforms.shape != (B, n + 1):
        raise TypeError(f"uniforms must be float32 ({B}, {n + 1})")
    if counts is not None and (counts.dtype != torch.int32 or counts.shape != (B,)):
        raise TypeError(f"counts must be int32 ({B},)")
    dev = target.device
    if dev.type != "cuda" or tokens.device != dev or uniforms.device != dev or \
            draft is not None and draft.device != dev or counts is not None and counts.device != dev:
        raise ValueError("all operands must be on one ROCm device (tensor.device.type == 'cuda')")
    target, p_sb, p_sr = _rows(target)
    q_sb = q_sr = 0
    if draft is not None:
        draft, q_sb, q_sr = _rows(draft)
    if uniforms.is_neg():
        uniforms = uniforms.resolve_neg()
    if n > 1 and tokens.stride(1) != 1:
        tokens = tokens.contiguous()
    if n > 0 and uniforms.stride(1) != 1:
        uniforms = uniforms.contiguous()
    if counts is not None and not counts.is_contiguous():
        counts = counts.contiguous()
    with nat.on_device(dev):
        out = torch.empty(B, n + 1, dtype=torch.int64, device=dev)
        accepted = torch.empty(B, dtype=torch.int64, device=dev)
        size = nat.sized("pp_verify_drafts_workspace_size", dev.index, B, V)
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        done, key = nat.zero_workspace(dev, 4 * B)
        rc = nat.lib().pp_verify_drafts(target.data_ptr(), p_sb, p_sr,
                                        draft.data_ptr() if draft is not None and n else None, q_sb, q_sr,
                                        _PROBABILITIES[target.dtype], B, n, V, tokens.data_ptr() if n else None,
                                        tokens.stride(0), uniforms.data_ptr(), uniforms.stride(0),
                                        counts.data_ptr() if counts is not None else None, out.data_ptr(),
                                        accepted.data_ptr(), ws.data_ptr() if size else None, size,
                                        done.data_ptr() if done is not None else None, 4 * B, nat.raw_stream(dev))
        if rc:
            nat.drop_workspace(key)
        nat.check(rc, "pp_verify_drafts")
    return Verified(out, accepted)
