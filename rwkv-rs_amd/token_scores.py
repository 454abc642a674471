"""What a language model's answer is scored by, on the gfx950 kernels of
include/rwkv_token_scores.h: the log probability of given tokens, the entropy
and the most likely alternatives of each row of logits, as one torch autograd
Function. All three have a gradient: of the log probability for training on
sampled answers, of the entropy for keeping them varied, of the alternatives'
log probabilities for learning from a teacher's. There is no second derivative and
no forward mode.

The forward reads the logits once, in their dtype, and keeps three numbers a row;
the backward reads them once more and writes their gradient once. Operands live
on the GPU; there is no CPU path.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .neighbors import _code, _no_tangent, _ptr, _stream

MAX_TOP = 64     # RWKV_TOKEN_SCORES_MAX_TOP


class TokenScores(NamedTuple):
    """Each of the logits' leading shape, the last two with ``top`` columns,
    the most likely first. float32, the ids int64."""
    log_prob: torch.Tensor
    entropy: torch.Tensor
    top_log_probs: torch.Tensor
    top_ids: torch.Tensor


def check_top(top: int, vocab: int) -> None:
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be 0 to {min(MAX_TOP, vocab)}, got {top}")


def _forward(logits, tokens, top, keep):
    """The four outputs and, with ``keep``, what the backward needs of each row."""
    rows, vocab = logits.shape
    dev = logits.device
    code = _code(logits.dtype)

    def row():
        return torch.empty(rows, dtype=torch.float32, device=dev)
    log_prob, entropy = row(), row()
    row_max, log_sum = (row(), row()) if keep else (None, None)
    top_lp = torch.empty(rows, top, dtype=torch.float32, device=dev)
    top_ids = torch.empty(rows, top, dtype=torch.int64, device=dev)
    _native.check(_native.lib().rwkv_token_scores_forward(
        logits.data_ptr(), tokens.data_ptr(), rows, vocab, top, code, log_prob.data_ptr(),
        entropy.data_ptr(), _ptr(row_max), _ptr(log_sum), top_lp.data_ptr(), top_ids.data_ptr(),
        _stream(dev)))
    return log_prob, entropy, top_lp, top_ids, row_max, log_sum


class _TokenScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top):
        log_prob, entropy, top_lp, top_ids, row_max, log_sum = _forward(logits, tokens, top, True)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(top_ids)
        ctx.save_for_backward(logits, tokens, row_max, log_sum, entropy, top_ids)
        return log_prob, entropy, top_lp, top_ids

    @staticmethod
    @once_differentiable
    def backward(ctx, d_log_prob, d_entropy, d_top, _):
        if d_log_prob is None and d_entropy is None and d_top is None:
            return None, None, None
        logits, tokens, row_max, log_sum, entropy, top_ids = ctx.saved_tensors
        rows, vocab = logits.shape
        grads = [None if g is None else g.to(torch.float32).contiguous()
                 for g in (d_log_prob, d_entropy, d_top)]
        dlogits = torch.empty_like(logits)
        _native.check(_native.lib().rwkv_token_scores_backward(
            logits.data_ptr(), tokens.data_ptr(), row_max.data_ptr(), log_sum.data_ptr(),
            entropy.data_ptr(), top_ids.data_ptr(), *(_ptr(g) for g in grads), rows, vocab, top_ids.shape[1],
            _code(logits.dtype), dlogits.data_ptr(), _stream(logits.device)))
        return dlogits, None, None


def token_scores(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenScores:
    """Scores of ``tokens`` ([...], integers) under ``logits`` ([..., vocab],
    fp32 or bf16), with the ``top`` (0 to 64) most likely alternatives of each
    row: the largest logits, the lower id first among equals.

    A token that a mask of minus infinity leaves out has log probability minus
    infinity. A row without a distribution (all of it masked, or a NaN or plus
    infinity in it) gets NaN, and -1 for its ids; a token outside [0, vocab) a
    NaN log probability."""
    if not logits.is_cuda or tokens.device != logits.device:
        raise ValueError("logits and tokens must be on the same GPU")
    if logits.dim() < 1 or tokens.shape != logits.shape[:-1]:
        raise ValueError("logits must be [..., vocab] and tokens [...]")
    if tokens.is_floating_point() or tokens.is_complex() or tokens.dtype == torch.bool:
        raise TypeError(f"tokens must be integers, got {tokens.dtype}")
    vocab = logits.shape[-1]
    check_top(top, vocab)
    if vocab == 0:
        raise ValueError("the vocabulary is empty")
    _no_tangent(logits, "token scores")
    lead = tokens.shape
    flat = logits if logits.dim() == 2 else logits.reshape(-1, vocab)
    if len(lead) != 1:
        tokens = tokens.reshape(-1)
    tokens = tokens.to(torch.int64).contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        out = _TokenScores.apply(flat.contiguous(), tokens, int(top))
    else:
        out = _forward(flat.contiguous(), tokens, int(top), False)[:4]
    if len(lead) != 1:
        out = [t.reshape(lead + t.shape[1:]) for t in out]
    return TokenScores(*out)
