"""The language model's training loss on the gfx950 kernels of
include/rwkv_lm_loss.h: l2wrap followed by the mean cross entropy of the
next-token logits (examples/rwkv-lm/src/model.rs:158-169), as one torch
autograd Function.

The forward reads the logits once (online maximum and log-sum-exp per row)
and keeps four numbers per row; the backward reads them once more and
writes the logits' gradient once, with l2wrap's term (kernels/l2wrap/mod.rs:
38-66: 1e-4 / num_tokens * max(logits) at each row's argmax) folded in. The
logits stay in their dtype (bf16 under autocast) instead of being cast to
fp32. Operands live on the GPU; there is no CPU path.

``linear_cross_entropy_l2wrap`` is the same loss straight from the last hidden
states and the unembedding (include/rwkv_linear_loss.h): the logits are formed in
tiles, twice, and neither they nor their gradient are ever whole in memory.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .neighbors import _code, _no_tangent, _on, _ptr, _stream

L2WRAP_FACTOR = 1e-4     # kernels/l2wrap/mod.rs:61-62
IGNORE_INDEX = -100      # a target that is not learned, as torch's cross entropy has it


class _CrossEntropyL2Wrap(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, num_tokens, ignore_index):
        rows, vocab = logits.shape
        dev = logits.device
        loss, lse, mx = (torch.empty(rows, dtype=torch.float32, device=dev) for _ in range(3))
        arg = torch.empty(rows, dtype=torch.int32, device=dev)
        name, ignore = _form(ignore_index)
        _native.call(name + "_forward", _ptr(logits), _ptr(targets), rows,
                     vocab, _code(logits.dtype), *ignore, _ptr(loss), _ptr(lse), _ptr(mx), _ptr(arg),
                     _stream(dev))
        ctx.save_for_backward(logits, targets, lse, mx, arg)
        ctx.ignore_index = ignore_index
        ctx.scale = L2WRAP_FACTOR / num_tokens if num_tokens > 0 else 0.0
        return loss

    @staticmethod
    def backward(ctx, dloss):
        logits, targets, lse, mx, arg = ctx.saved_tensors
        rows, vocab = logits.shape
        g = dloss.to(torch.float32).contiguous()
        dlogits = torch.empty_like(logits)
        name, ignore = _form(ctx.ignore_index)
        _native.call(name + "_backward", _ptr(logits), _ptr(targets), _ptr(lse),
                     _ptr(mx), _ptr(arg), _ptr(g), float(ctx.scale), rows, vocab,
                     _code(logits.dtype), *ignore, _ptr(dlogits), _stream(logits.device))
        return dlogits, None, None, None


def _form(ignore_index):
    """The entry points' name and their further argument."""
    if ignore_index is None:
        return "rwkv_cross_entropy_l2wrap", ()
    return "rwkv_cross_entropy_l2wrap_ignore", (ignore_index,)


def cross_entropy_l2wrap_rows(logits: torch.Tensor, targets: torch.Tensor,
                              num_tokens: int, ignore_index: Optional[int] = None) -> torch.Tensor:
    """Per-row cross entropy of ``logits`` ([rows, vocab], fp32 or bf16) against ``targets`` ([rows] integer), with l2wrap's
    gradient term for ``num_tokens`` tokens in the backward. A target outside
    [0, vocab) gives its row a NaN loss, but for ``ignore_index``, where one is given: such
    a row has loss 0 and no gradient, whatever its logits are."""
    if not logits.is_cuda or not targets.is_cuda:
        raise ValueError("logits and targets must be GPU tensors")
    if logits.dim() != 2 or targets.shape != (logits.shape[0],):
        raise ValueError("logits must be [rows, vocab] and targets [rows]")
    return _CrossEntropyL2Wrap.apply(logits.contiguous(), targets.to(torch.int64).contiguous(),
                                     int(num_tokens), None if ignore_index is None else int(ignore_index))


def cross_entropy_l2wrap(logits: torch.Tensor, targets: torch.Tensor,
                         ignore_index: Optional[int] = None) -> torch.Tensor:
    """``F.cross_entropy(l2wrap(logits, rows), targets)``: the mean over the
    rows, l2wrap counting every row as a token (model.rs:161-169). With an
    ``ignore_index`` over those whose target it is not (0 when there is none)."""
    rows = cross_entropy_l2wrap_rows(logits, targets, logits.shape[0], ignore_index)
    return rows.mean() if ignore_index is None else _mean_of_learned(rows, targets, ignore_index)


def _mean_of_learned(rows, targets, ignore_index):
    # in 64 bits: a narrow type would be compared with ignore_index cut off to it
    return rows.sum() / (targets.to(torch.int64) != ignore_index).sum().clamp(min=1)


# ------------------------------------------- from hidden states and unembedding
def _workspace(nbytes: int, device) -> torch.Tensor:
    if nbytes < 0:
        raise ValueError("hidden states or an unembedding of this size are not supported")
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _linear_forward(hidden, weight, targets, ignore_index):
    """Every row's loss, and what the backward needs of it: a [3, rows] tensor of the logarithm
    of its exponentials' sum over its maximum, that maximum and (as int32) its argmax."""
    (rows, c), vocab, dev = hidden.shape, weight.shape[0], hidden.device
    code, lib = _code(hidden.dtype), _native.lib()
    nbytes = lib.rwkv_linear_loss_forward_workspace_bytes(rows, vocab, c, code)
    ws = _workspace(nbytes, dev)
    loss = torch.empty(rows, dtype=torch.float32, device=dev)
    kept = torch.empty(3, rows, dtype=torch.float32, device=dev)
    at = kept.data_ptr()
    with _on(dev):
        _native.check(lib.rwkv_linear_loss_forward(
            hidden.data_ptr(), weight.data_ptr(), targets.data_ptr(), rows, vocab, c, code, ignore_index,
            loss.data_ptr(), at, at + 4 * rows, at + 8 * rows, ws.data_ptr(), nbytes, _stream(dev)))
    return loss, kept


class _LinearCrossEntropyL2Wrap(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, num_tokens, ignore_index):
        loss, kept = _linear_forward(hidden, weight, targets, ignore_index)
        ctx.save_for_backward(hidden, weight, targets, kept)
        ctx.scale = L2WRAP_FACTOR / num_tokens if num_tokens > 0 else 0.0
        ctx.ignore_index = ignore_index
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        hidden, weight, targets, kept = ctx.saved_tensors
        (rows, c), vocab, dev = hidden.shape, weight.shape[0], hidden.device
        code, at, lib = _code(hidden.dtype), kept.data_ptr(), _native.lib()
        g = dloss if dloss.is_contiguous() else dloss.contiguous()
        need = ctx.needs_input_grad
        dhidden = torch.empty_like(hidden) if need[0] else None
        dweight = torch.empty_like(weight) if need[1] else None
        nbytes = lib.rwkv_linear_loss_backward_workspace_bytes(rows, vocab, c, code)
        ws = _workspace(nbytes, dev)
        with _on(dev):
            _native.check(lib.rwkv_linear_loss_backward(
                hidden.data_ptr(), weight.data_ptr(), targets.data_ptr(), at, at + 4 * rows, at + 8 * rows,
                g.data_ptr(), ctx.scale, rows, vocab, c, code, ctx.ignore_index, _ptr(dhidden), _ptr(dweight),
                ws.data_ptr(), nbytes, _stream(dev)))
        return dhidden, dweight, None, None, None


def _operand(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def linear_cross_entropy_l2wrap_rows(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                                     num_tokens: int, ignore_index: int = IGNORE_INDEX) -> torch.Tensor:
    """``cross_entropy_l2wrap_rows(hidden @ weight.T, targets, num_tokens)`` without
    the logits: ``hidden`` [rows, c] and ``weight`` [vocab, c] are both float32 or both
    bfloat16, and differentiable once, in reverse mode. Logits are not rounded on the
    way. A row whose target is ``ignore_index`` has loss 0 and no gradient, whatever its
    hidden state is; one whose target is otherwise outside [0, vocab) a NaN loss."""
    if not hidden.is_cuda or weight.device != hidden.device or targets.device != hidden.device:
        raise ValueError("hidden, weight and targets must be on the same GPU")
    if hidden.dim() != 2 or weight.dim() != 2 or weight.shape[1] != hidden.shape[1] \
            or targets.shape != hidden.shape[:1]:
        raise ValueError("hidden must be [rows, c], weight [vocab, c] and targets [rows]")
    if 0 in weight.shape:
        raise ValueError("the vocabulary or the hidden states are empty")
    if weight.dtype != hidden.dtype:
        raise TypeError(f"hidden and weight must have one dtype, got {hidden.dtype} and {weight.dtype}")
    if targets.is_floating_point() or targets.is_complex() or targets.dtype == torch.bool:
        raise TypeError(f"targets must be integers, got {targets.dtype}")
    _code(hidden.dtype)
    for t in (hidden, weight):
        _no_tangent(t, "losses from hidden states")
    hidden, weight = _operand(hidden), _operand(weight)
    targets = targets.to(torch.int64).contiguous()
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _LinearCrossEntropyL2Wrap.apply(hidden, weight, targets, int(num_tokens), int(ignore_index))
    return _linear_forward(hidden, weight, targets, int(ignore_index))[0]


def linear_cross_entropy_l2wrap(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                                ignore_index: int = IGNORE_INDEX) -> torch.Tensor:
    """``cross_entropy_l2wrap(hidden @ weight.T, targets)`` without the logits: the
    mean over the rows that are not ignored (0 when all are), l2wrap counting every
    row as a token."""
    rows = linear_cross_entropy_l2wrap_rows(hidden, weight, targets, hidden.shape[0], ignore_index)
    return _mean_of_learned(rows, targets, ignore_index)
