"""What a step's logits answer: log probabilities of given tokens, entropy, alternatives."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native as nat

TOP_MAX = 64
_LOGITS = {torch.float16: nat.PP_F16, torch.bfloat16: nat.PP_BF16, torch.float32: nat.PP_F32}


class TokenLogprobs(NamedTuple):
    """float32 ``logprob`` (of ``tokens``' shape) and ``entropy`` (rows,); with ``top`` alternatives
    int64 ``top_ids`` and float32 ``top_logprobs`` (rows, top), otherwise None."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]


def token_logprobs(logits, tokens, *, top=0):
    """Log probabilities under ``logits`` (rows, V), float16, bfloat16 or float32, in one pass.

    ``tokens`` int64 (rows,) or (rows, n): ``logprob = x[token] - log sum e^x``, NaN for a token outside
    [0, V).  ``entropy = log sum e^x - sum p x``.  ``top`` (at most 64): the largest logits in order,
    equal ones by the lower index.  A logit of -inf has probability 0; a row of nothing else, or one
    that holds a NaN or +inf, gives NaN.  Sums are held in float32.  There is no backward pass: the results
    carry no gradient, whether ``logits`` asks for one or not.
    """
    if logits.dim() != 2 or logits.dtype not in _LOGITS:
        raise TypeError("logits must be float16, bfloat16 or float32 (rows, V)")
    rows, V = logits.shape
    if tokens.dtype != torch.int64 or tokens.dim() not in (1, 2) or tokens.shape[0] != rows:
        raise TypeError("tokens must be int64 (rows,) or (rows, n)")
    dev = logits.device
    if dev.type != "cuda" or tokens.device != dev:
        raise ValueError("logits and tokens must be on one ROCm device (tensor.device.type == 'cuda')")
    if V < 1:
        raise ValueError("a row needs a logit")
    if not 0 <= top <= min(TOP_MAX, V):
        raise ValueError(f"top must be in 0..{min(TOP_MAX, V)}")
    if logits.is_neg():                              # memory that holds the values negated
        logits = logits.resolve_neg()
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    per_row = 1 if tokens.dim() == 1 else tokens.shape[1]
    if tokens.dim() == 2 and per_row > 1 and tokens.stride(1) != 1:
        tokens = tokens.contiguous()
    with nat.on_device(dev):
        stats = torch.empty(rows * (per_row + 1 + top), dtype=torch.float32, device=dev)
        lp, entropy, tl = stats.split([rows * per_row, rows, rows * top])
        ids = torch.empty((rows, top), dtype=torch.int64, device=dev) if top else None
        size = nat.sized("pp_logprobs_workspace_size", dev.index, rows, V, top)
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        nat.check(nat.lib().pp_logprobs(logits.data_ptr(), logits.stride(0), _LOGITS[logits.dtype], rows, V,
                                        tokens.data_ptr(), tokens.stride(0), per_row, top, lp.data_ptr(),
                                        entropy.data_ptr(), ids.data_ptr() if top else None,
                                        tl.data_ptr() if top else None, ws.data_ptr() if size else None, size,
                                        nat.raw_stream(dev)), "pp_logprobs")
    return TokenLogprobs(lp.view(tokens.shape), entropy, ids, tl.view(rows, top) if top else None)
