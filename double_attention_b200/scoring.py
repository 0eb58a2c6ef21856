"""Scores of tokens under a model's logits: log probabilities, entropies and top alternatives, with a backward pass.

:func:`token_log_probs` reads the logits once and keeps nothing of their size; its backward pass reads them once more
and writes their gradient.  ``DoubleAttentionLM.score`` and ``Int8DoubleAttentionLM.score`` call it.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from ._lib import ptr
from .eight_bit import _CODES, _FirstOrder, _device_of, _host, _launch, _new, _rows

IGNORE = -100   # a token that is none
MAX_TOP = 32


class TokenLogProbs(NamedTuple):
    """Scores of tokens [...] under logits [..., V].

    log_probs: fp32 [...], the tokens' log probabilities (0 for the token -100).
    entropy: fp32 [...], -sum p log p of each row.
    top_log_probs, top_tokens: fp32 and int64 [..., top], the largest first, of equal ones the lowest token; None without
        ``top``.
    """

    log_probs: Tensor
    entropy: Tensor
    top_log_probs: Tensor | None
    top_tokens: Tensor | None


def _forward(logits: Tensor, tokens: Tensor, top: int, device: int, keep: bool):
    lead, v = logits.shape[:-1], logits.shape[-1]
    x, rows, ld = _rows(logits)
    made = _new(lead, torch.float32, logits.device), _new(lead, torch.float32, logits.device)
    top_lp = top_tokens = stats = None
    if top:
        top_lp = torch.empty(*lead, top, dtype=torch.float32, device=logits.device)
        top_tokens = torch.empty(*lead, top, dtype=torch.int64, device=logits.device)
    if keep:
        stats = _new((rows, 2), torch.float32, logits.device)
    if rows:
        _launch(device, "da_token_log_probs", x.data_ptr(), _CODES[logits.dtype], ld, rows, v, tokens.data_ptr(), top,
                made[0].data_ptr(), made[1].data_ptr(), ptr(top_lp), ptr(top_tokens), ptr(stats))
    return *made, top_lp, top_tokens, stats


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: Tensor, tokens: Tensor, top: int, device: int):  # type: ignore[override]
        log_probs, entropy, top_lp, top_tokens, stats = _forward(logits, tokens, top, device, True)
        ctx.save_for_backward(logits, tokens, stats, entropy)
        ctx.device = device
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_lp, top_tokens)
        return log_probs, entropy, top_lp, top_tokens

    @staticmethod
    def backward(ctx, d_log_probs, d_entropy, _top_lp, _top_tokens):  # type: ignore[override]
        first = d_entropy if d_log_probs is None else d_log_probs
        if first is None:
            return None, None, None, None
        with torch.no_grad():
            d = _TokenLogProbs._gradient(ctx, d_log_probs, d_entropy)
        if torch.is_grad_enabled():  # create_graph: raises when differentiated again
            d = _FirstOrder.apply(d.requires_grad_(), first, "token_log_probs")
        return d, None, None, None

    @staticmethod
    def _gradient(ctx, d_log_probs: Tensor | None, d_entropy: Tensor | None) -> Tensor:
        logits, tokens, stats, entropy = ctx.saved_tensors
        x, rows, ld = _rows(logits)
        v = logits.shape[-1]
        g = None if d_log_probs is None else d_log_probs.float().contiguous()
        h = None if d_entropy is None else d_entropy.float().contiguous()
        d = _new(logits.shape, logits.dtype, logits.device)
        if rows:
            _launch(ctx.device, "da_token_log_probs_bwd", x.data_ptr(), _CODES[logits.dtype], ld, rows, v, tokens.data_ptr(),
                    stats.data_ptr(), entropy.data_ptr(), ptr(g), ptr(h), d.data_ptr(), v)
        return d


def token_log_probs(logits: Tensor, tokens: Tensor, *, top: int = 0) -> TokenLogProbs:
    """Log probabilities of ``tokens`` [...] under ``logits`` [..., V], each row's entropy, and its ``top`` likeliest tokens.

    logits in fp32, bf16 or fp16, any strides; all sums in fp32.  Entries of minus infinity have probability 0; a row
    with a NaN, with plus infinity or with no finite entry is NaN.  A token of -100 has log probability 0 and passes no
    gradient, whatever its row holds; any other outside [0, V) is NaN.  ``top`` at most 32; NaN comes before numbers there.

    Differentiable in ``logits`` through ``log_probs`` and ``entropy`` (the alternatives carry no gradient)."""
    name = "token_log_probs"
    if logits.is_cuda:
        done = _host().score(logits, tokens, top)
        if done is not None:
            return TokenLogProbs(*done)
    if logits.dtype not in _CODES:
        raise ValueError(f"{name} takes logits in float32, bfloat16 or float16, got {logits.dtype}")
    if not logits.ndim or not logits.shape[-1] or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"{name} takes logits [..., V] with V at least 1 and tokens [...], got {tuple(logits.shape)} and "
                         f"{tuple(tokens.shape)}")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{name} takes tokens in int64 or int32, got {tokens.dtype}")
    if not 0 <= top <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError(f"{name} gives 0 to {min(MAX_TOP, logits.shape[-1])} alternatives here, asked for {top}")
    device = _device_of(name, logits, tokens)
    tokens = tokens.long().contiguous()
    if torch.is_grad_enabled() and logits.requires_grad or torch.autograd.forward_ad._current_level >= 0:
        return TokenLogProbs(*_TokenLogProbs.apply(logits, tokens, top, device))
    return TokenLogProbs(*_forward(logits, tokens, top, device, False)[:4])
