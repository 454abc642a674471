"""Dropout on the gfx950 kernel of include/rwkv_dropout.h: the mask comes from a
counter-based generator and is drawn again in the backward instead of being
stored. ``dropout_add`` adds the result to a residual stream in the same pass.

``rng`` is an int64 tensor [seed, step] on the GPU: a training step counts the
second number up, and the calls within a step take different sites. Element i's
fate depends on seed, step, site and i alone, not on the type, the GPU or the
launch, and ``keep_mask`` says it in plain torch, on any device. An rng that is changed in
place between a forward and its backward is refused by autograd; give each forward
a clone where that may happen.
"""

from __future__ import annotations

import torch

from . import _native
from .neighbors import _code, _on, _ptr, _stream

LOW32 = 0xFFFFFFFF


def _check(x: torch.Tensor, p: float, rng: torch.Tensor, site: int) -> None:
    if rng.dtype != torch.int64 or rng.shape != (2,) or rng.device != x.device:
        raise ValueError("rng must be an int64 tensor [seed, step] on the operands' device")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be 0 to 1, got {p}")
    if not 0 <= site <= LOW32:
        raise ValueError(f"site must be 0 to 2^32 - 1, got {site}")


def _run(x, residual, rng, site, p, code, out_dtype, out_code):
    """Of contiguous operands. The codes are the dtypes'."""
    dev = x.device
    out = torch.empty_like(x, dtype=out_dtype)
    with _on(dev):
        _native.check(_native.lib().rwkv_dropout(
            x.data_ptr(), _ptr(residual), rng.data_ptr(), site, p, x.numel(), code, out_code,
            out.data_ptr(), _stream(dev)))
    return out


class _Dropout(torch.autograd.Function):
    """x to ``out_dtype``. Its backward is itself, the other way round."""

    @staticmethod
    def forward(ctx, x, rng, site, p, code, out_dtype, out_code):
        ctx.save_for_backward(rng)
        ctx.args = site, p, out_code, x.dtype, code
        return _run(x, None, rng, site, p, code, out_dtype, out_code)

    @staticmethod
    def backward(ctx, grad):
        return _backward(ctx, grad), None, None, None, None, None, None


def _backward(ctx, grad):
    rng, = ctx.saved_tensors
    if torch.is_grad_enabled():        # a gradient of the gradient is wanted
        return _Dropout.apply(grad.contiguous(), rng, *ctx.args)
    return _run(grad if grad.is_contiguous() else grad.contiguous(), None, rng, *ctx.args)


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, x, rng, site, p, code, out_code):
        ctx.save_for_backward(rng)
        ctx.args = site, p, out_code, x.dtype, code
        return _run(x, residual, rng, site, p, code, residual.dtype, out_code)

    @staticmethod
    def backward(ctx, grad):
        return grad, _backward(ctx, grad) if ctx.needs_input_grad[1] else None, None, None, None, None, None


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor, site: int = 0) -> torch.Tensor:
    """``x`` (float32 or bfloat16) with each element zeroed with probability ``p``,
    rounded to a multiple of 2^-16, and the others divided by 1 - p. Differentiable
    in ``x``. A dropped element is 0 even where x is NaN or infinite."""
    if not x.is_cuda:
        raise ValueError("x must be a GPU tensor")
    code = _code(x.dtype)
    _check(x, p, rng, site)
    return _Dropout.apply(x.contiguous(), rng.contiguous(), int(site), float(p), code, x.dtype, code)


def dropout_add(residual: torch.Tensor, x: torch.Tensor, p: float, rng: torch.Tensor,
                site: int = 0) -> torch.Tensor:
    """``residual + dropout(x, p, rng, site)`` in one pass, summed in float32 and
    rounded once to the residual's dtype; ``x`` may have another one. Differentiable
    in both."""
    if not x.is_cuda or residual.device != x.device:
        raise ValueError("residual and x must be on the same GPU")
    if residual.shape != x.shape:
        raise ValueError(f"residual and x must have one shape, got {tuple(residual.shape)} and {tuple(x.shape)}")
    code, out_code = _code(x.dtype), _code(residual.dtype)
    _check(x, p, rng, site)
    return _DropoutAdd.apply(residual.contiguous(), x.contiguous(), rng.contiguous(), int(site), float(p),
                             code, out_code)


def keep_probability(p: float) -> float:
    """1 - p as it is used: a multiple of 2^-16."""
    return round((1.0 - p) * 65536) / 65536


def _philox(c0, c1, c2, c3, seed):
    """Philox4x32-10 of the counters c0 .. c3 and the key ``seed`` (int64 tensors, the
    former below 2^32): four words."""
    c = [c0, c1, c2, c3]
    k = [seed & LOW32, (seed >> 32) & LOW32]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57     # modulo 2^64: the shift's sign bits are masked off
        c = [((b >> 32) & LOW32) ^ c[1] ^ k[0], b & LOW32, ((a >> 32) & LOW32) ^ c[3] ^ k[1], a & LOW32]
        k = [(k[0] + 0x9E3779B9) & LOW32, (k[1] + 0xBB67AE85) & LOW32]
    return c


def keep_mask(shape, p: float, rng: torch.Tensor, site: int = 0) -> torch.Tensor:
    """The elements that ``dropout`` of a tensor of this shape keeps, as a bool tensor
    on ``rng``'s device, in plain torch."""
    _check(rng, p, rng, site)
    n = torch.Size(shape).numel()
    q = torch.arange(-(-n // 8), device=rng.device)
    step = (rng[1] & LOW32).expand_as(q)
    words = torch.stack(_philox(q & LOW32, q >> 32, torch.full_like(q, site), step, rng[0]), dim=1)
    numbers = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)[:n].reshape(shape)
    return numbers < round((1.0 - p) * 65536)
