"""Log probabilities of given tokens, with the entropy and top alternatives.

The engine's sampler (``engine/sampler.py``) takes the argmax of the logits; a
server also answers how likely the chosen tokens were and what stood next to
them.  :func:`b200_token_logprobs` reads each row of logits once
(``b200mm_token_logprobs``).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _capi

MAX_TOP = 64


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # (...) float32
    entropy: torch.Tensor       # (...) float32, natural logarithm
    top_ids: torch.Tensor       # (..., top) int64
    top_logprobs: torch.Tensor  # (..., top) float32


def b200_token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenLogprobs:
    """``log_softmax(logits)[tokens]``, the rows' entropy, and their ``top``
    most likely tokens (descending; equal logits by ascending id).

    Args:
        logits: (..., V), float32, float16 or bfloat16 on a CUDA device.
        tokens: (...) int64 on the same device; one outside [0, V) gets NaN.
        top: alternatives per row, at most ``min(V, 64)``.

    Sums are fp32.  -inf logits are tokens of probability 0; a row with a NaN
    or +inf, or with nothing but -inf, gets NaN (its ids stay ordered, NaN first).
    """
    if logits.dim() < 1 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens {tuple(tokens.shape)} must be logits' shape {tuple(logits.shape)} without the last dim")
    if tokens.dtype != torch.int64:
        raise ValueError(f"tokens must be int64, got {tokens.dtype}")
    if tokens.device != logits.device:
        raise ValueError(f"logits ({logits.device}) and tokens ({tokens.device}) must be on the same device")
    V = logits.shape[-1]
    if V < 1 or not 0 <= top <= min(V, MAX_TOP):
        raise ValueError(f"top must be in 0..{min(V, MAX_TOP)}, got {top}")
    code = _capi.dtype_code(logits.dtype)
    _capi.require_cuda(logits)
    x = logits if logits.dim() == 2 else logits.reshape(-1, V)
    if x.stride(-1) != 1 or x.stride(0) < V:
        x = x.contiguous()
    M = x.shape[0]
    lead = logits.shape[:-1]
    toks = tokens if tokens.is_contiguous() else tokens.contiguous()
    lp = x.new_empty(lead, dtype=torch.float32)
    ent, ids = torch.empty_like(lp), toks.new_empty((*lead, top))
    lps = lp.new_empty((*lead, top))
    if M:
        _capi.launch("b200mm_token_logprobs", x, x.data_ptr(), x.stride(0) if M > 1 else V, toks.data_ptr(), lp.data_ptr(), ent.data_ptr(),
                     ids.data_ptr(), lps.data_ptr(), M, V, top, code)
    return TokenLogprobs(lp, ent, ids, lps)
