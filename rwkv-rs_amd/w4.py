"""Linear layers with 4-bit weights on the gfx950 kernels of include/rwkv_w4.h,
for serving: a step of a few sequences reads every weight once, so it takes
as long as their bytes do.

* ``quantize``       a weight matrix [out, in] to 4-bit floats (0, 0.5, 1, 1.5,
                     2, 3, 4, 6 with a sign) with a bf16 scale for each group
                     of 32, 64 or 128 inputs
* ``dequantize``     the matrix that they stand for
* ``linear``         rows of activations times it
* ``W4Linear``       a module in the place of a bias-free ``nn.Linear``
* ``quantize_model`` a model's projections and unembedding, in place

There are no gradients: the products are for serving, and refuse operands that
ask for one or carry a forward-mode tangent. Operands live on the GPU; there is no CPU path.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn as nn

from . import _native
from .neighbors import _code, _no_tangent, _ptr, _stream

GROUPS = (32, 64, 128)
MAX_DIM = 1 << 26        # RWKV_W4_MAX_DIM
FEW_ROWS = 16            # up to as many rows no workspace is asked for


@dataclass(frozen=True)
class W4Weight:
    """A quantised [out_features, in_features] matrix, in include/rwkv_w4.h's
    layout: ``packed`` uint8 [ceil(out / 16), ceil(in / 128), 4, 16, 16] and
    ``scales`` bfloat16 [ceil(out / 16), ceil(in / 128), 16, 128 / group_size]."""
    packed: torch.Tensor
    scales: torch.Tensor
    out_features: int
    in_features: int
    group_size: int

    def __post_init__(self):
        _check_sizes(self.out_features, self.in_features, self.group_size)
        n, k = -(-self.out_features // 16), -(-self.in_features // 128)
        if self.packed.dtype != torch.uint8 or self.packed.shape != (n, k, 4, 16, 16):
            raise ValueError(f"packed must be uint8 [{n}, {k}, 4, 16, 16]")
        if self.scales.dtype != torch.bfloat16 or self.scales.shape != (n, k, 16, 128 // self.group_size):
            raise ValueError(f"scales must be bfloat16 [{n}, {k}, 16, {128 // self.group_size}]")
        if self.packed.device != self.scales.device:
            raise ValueError("packed and scales must be on one device")
        if not self.packed.is_contiguous() or not self.scales.is_contiguous():
            raise ValueError("packed and scales must be contiguous")


def _check_sizes(out_features: int, in_features: int, group_size: int) -> None:
    if group_size not in GROUPS:
        raise ValueError(f"group_size must be one of {GROUPS}, got {group_size}")
    if not 0 < out_features <= MAX_DIM or not 0 < in_features <= MAX_DIM:
        raise ValueError(f"a weight has 1 to {MAX_DIM} outputs and inputs")


def quantize(weight: torch.Tensor, group_size: int = 64) -> W4Weight:
    """``weight`` ([out, in], fp32 or bf16) as 4-bit floats with a scale for
    every ``group_size`` inputs of an output. A group that holds an infinity
    or a NaN gets a NaN scale."""
    if not weight.is_cuda:
        raise ValueError("weight must be a GPU tensor")
    if weight.dim() != 2:
        raise ValueError("weight must be [out, in]")
    out, d_in = weight.shape
    _check_sizes(out, d_in, group_size)
    code = _code(weight.dtype)
    w = weight.detach().contiguous()
    n, k = -(-out // 16), -(-d_in // 128)
    packed = torch.empty(n, k, 4, 16, 16, dtype=torch.uint8, device=w.device)
    scales = torch.empty(n, k, 16, 128 // group_size, dtype=torch.bfloat16, device=w.device)
    _native.call("rwkv_w4_quantize", w.data_ptr(), out, d_in, group_size, code, packed.data_ptr(),
                 scales.data_ptr(), _stream(w.device))
    return W4Weight(packed, scales, out, d_in, group_size)


def dequantize(weight: W4Weight, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The [out, in] matrix ``weight`` stands for: exact in fp32, rounded in bf16."""
    dev = weight.packed.device
    if dev.type != "cuda":
        raise ValueError("weight must be on the GPU")
    code = _code(dtype)
    out = torch.empty(weight.out_features, weight.in_features, dtype=dtype, device=dev)
    _native.call("rwkv_w4_dequantize", weight.packed.data_ptr(), weight.scales.data_ptr(),
                 weight.out_features, weight.in_features, weight.group_size, code, out.data_ptr(),
                 _stream(dev))
    return out


def linear(x: torch.Tensor, weight: W4Weight) -> torch.Tensor:
    """``x`` ([..., in], fp32 or bf16) times the transpose of ``weight``:
    [..., out] in x's dtype, sums in fp32, rounded once."""
    dev = weight.packed.device
    if x.device != dev or dev.type != "cuda":
        raise ValueError("x and weight must be on the same GPU")
    if x.dim() < 1 or x.shape[-1] != weight.in_features:
        raise ValueError(f"x must be [..., {weight.in_features}]")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("products with 4-bit weights have no gradient (use torch.no_grad)")
    code = _code(x.dtype)
    _no_tangent(x, "products with 4-bit weights")
    x = x.contiguous()
    y = torch.empty(*x.shape[:-1], weight.out_features, dtype=x.dtype, device=dev)
    rows = x.numel() // weight.in_features
    lib = _native.lib()
    nbytes = 0
    ws = None
    if rows > FEW_ROWS:
        nbytes = lib.rwkv_w4_linear_workspace_bytes(rows, weight.out_features, weight.in_features, code)
        if nbytes > 0:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _native.check(lib.rwkv_w4_linear(
        x.data_ptr(), weight.packed.data_ptr(), weight.scales.data_ptr(), rows, weight.out_features,
        weight.in_features, weight.group_size, code, y.data_ptr(), _ptr(ws), nbytes, _stream(dev)))
    return y


class W4Linear(nn.Module):
    """A bias-free linear layer with a 4-bit weight, in the place of an
    ``nn.Linear`` of a model that is served. Under autocast x is cast to
    autocast's dtype, as ``nn.Linear`` does. Casting the module leaves its weight."""

    def __init__(self, weight: W4Weight):
        super().__init__()
        self.out_features, self.in_features = weight.out_features, weight.in_features
        self.group_size = weight.group_size
        self.register_buffer("packed", weight.packed)
        self.register_buffer("scales", weight.scales)

    @classmethod
    def from_linear(cls, module: nn.Linear, group_size: int = 64) -> "W4Linear":
        if module.bias is not None:
            raise ValueError("a linear layer with a bias is not taken")
        return cls(quantize(module.weight, group_size))

    @property
    def weight(self) -> W4Weight:
        return W4Weight(self.packed, self.scales, self.out_features, self.in_features, self.group_size)

    def _apply(self, fn, recurse=True):
        # a cast of the model (.float(), .half()) moves the buffers but leaves their
        # types, which are the format's
        before = self.packed, self.scales
        super()._apply(fn, recurse)
        for name, old in zip(("packed", "scales"), before):
            new = getattr(self, name)
            if new.dtype != old.dtype:
                setattr(self, name, old.to(new.device))
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if torch.is_autocast_enabled(x.device.type):
            x = x.to(torch.get_autocast_dtype(x.device.type))
        return linear(x, self.weight)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"group_size={self.group_size}")


def quantize_model(model: nn.Module, group_size: int = 64) -> nn.Module:
    """Replace every bias-free ``nn.Linear`` of ``model`` (an
    ``AutoRegressiveModel``'s projections, channel mixers and unembedding) by a
    ``W4Linear`` of its weight, in place; the embedding, the LoRAs and the norms
    stay as they are. Returns the model, which is then for serving only; where a
    layer is refused (its type, its device), none is replaced."""
    if isinstance(model, nn.Linear):
        raise ValueError("model must hold the linear layers, not be one")
    places = [(parent, name, child) for parent in list(model.modules())
              # named_children() leaves out a child's second name
              for name, child in parent._modules.items()
              if type(child) is nn.Linear and child.bias is None]
    done = {}
    for _, _, child in places:   # all of them before the model changes: one may be refused
        if child not in done:
            done[child] = W4Linear.from_linear(child, group_size)
    for parent, name, child in places:
        setattr(parent, name, done[child])
    return model
