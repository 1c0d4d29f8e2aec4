"""Log probabilities of given tokens, with entropy and the most likely alternatives.

``token_logprobs`` reads rows of logits once: with log Z the logarithm of a row's
sum of exponentials, log p(t) = x_t - log Z, the entropy is
H = -sum p log p, and the alternatives are the ``top`` largest logits (ties to
the lower id) with theirs.  All in fp32, whatever the logits' type.

-inf logits (tokens that are not allowed) have probability 0.  A row of nothing
else, or one with a NaN or +inf, has no distribution: all its numbers are NaN
(its ids are the order of its logits still, NaN above all).

On the GPU the work is this library's kernels (no fallback: the library must load); CPU
tensors take the formulas.  Inference only: logits that ask for a gradient are refused.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .q8 import INT_MAX, _asks_gradient, _call

MAX_TOP = 64
MAX_VOCAB = INT_MAX - 65536
MAX_ROWS = 2 ** 24 - 1
_KINDS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class TokenLogprobs(NamedTuple):
    """logprob and entropy [...] fp32; top_logprobs [..., top] fp32 and top_ids [..., top] int64."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_ids: torch.Tensor


def _formula(x: torch.Tensor, tokens: torch.Tensor, top: int) -> TokenLogprobs:
    x = x.float()
    vocab = x.shape[-1]
    lp = torch.log_softmax(x, dim=-1)
    odd = ~(x.amax(dim=-1).isfinite()) | x.isnan().any(dim=-1)
    lp = torch.where(odd.unsqueeze(-1), torch.full_like(lp, float("nan")), lp)
    entropy = -torch.where(lp == float("-inf"), torch.zeros_like(lp), lp.exp() * lp).sum(dim=-1)
    ok = (tokens >= 0) & (tokens < vocab)
    picked = lp.gather(-1, tokens.clamp(0, vocab - 1).unsqueeze(-1)).squeeze(-1)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top].contiguous()
    return TokenLogprobs(torch.where(ok, picked, torch.full_like(picked, float("nan"))), entropy, lp.gather(-1, ids), ids)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """logits [..., vocab] (float32, bfloat16 or float16), tokens [...] (integers; outside
    [0, vocab): NaN), up to 64 alternatives.

    Rows may lie apart (a column range of wider ones) and are read in place."""
    who = "token_logprobs"
    if logits.dim() < 1 or logits.dtype not in _KINDS:
        raise ValueError(f"{who}: logits must be float32, bfloat16 or float16 [..., vocab] "
                         f"(got {logits.dtype} {tuple(logits.shape)})")
    vocab = logits.shape[-1]
    lead = logits.shape[:-1]
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"{who}: the vocabulary has from 1 to {MAX_VOCAB} tokens (got {vocab})")
    if tokens.dtype not in (torch.int64, torch.int32) or tokens.shape != lead or tokens.device != logits.device:
        raise ValueError(f"{who}: tokens must be int64 (or int32) {tuple(lead)} on the logits' device "
                         f"(got {tokens.dtype} {tuple(tokens.shape)} on {tokens.device})")
    if isinstance(top, bool) or not isinstance(top, int) or not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"{who}: top must be a whole number from 0 to {min(MAX_TOP, vocab)} (got {top!r})")
    if _asks_gradient(logits):
        raise ValueError(f"{who}: the logits ask for a gradient, and this operator has none")
    rows = logits.numel() // vocab
    if rows > MAX_ROWS:
        raise ValueError(f"{who}: at most {MAX_ROWS} rows (got {rows})")
    if not logits.is_cuda:
        return _formula(logits, tokens.long(), top)
    device = logits.device
    if logits.dim() == 2 and logits.stride(1) == 1 or logits.is_contiguous():
        stride = logits.stride(0) if logits.dim() == 2 else vocab
    else:
        logits, stride = logits.contiguous(), vocab
    tokens = tokens.to(torch.int64).contiguous()
    out = torch.empty((2, *lead), dtype=torch.float32, device=device)
    top_lp = torch.empty((*lead, top), dtype=torch.float32, device=device)
    top_ids = torch.empty((*lead, top), dtype=torch.int64, device=device)
    result = TokenLogprobs(out[0], out[1], top_lp, top_ids)
    if rows:
        need = _lib.load().nkv_token_logprobs_workspace(rows, vocab, top)
        # (dropped behind the launch: the stream orders its reuse)
        ws = torch.empty(need, dtype=torch.float32, device=device) if need else None
        at = out.data_ptr()
        _call("token_logprobs", logits.get_device(), logits.data_ptr(), _KINDS[logits.dtype], stride, rows, vocab,
              tokens.data_ptr(), top, at, at + 4 * rows, top_lp.data_ptr(), top_ids.data_ptr(),
              ws.data_ptr() if need else None)
    return result


__all__ = ["TokenLogprobs", "token_logprobs"]
