"""The 8-bit baseline of the quantized layers: nn.Linear with int8 weights
(a scale per output channel) and int8 activations (a scale per token), for
inference.  Device tensors run rpfq_linear_int8; host tensors the same
arithmetic in torch.
"""
from __future__ import annotations

import torch
import torch.nn as nn


def quantize_rows(x: torch.Tensor):
    """(codes int8, scale float32) of the rows of x, as rpfq_quantize_int8
    defines them: rint(127 x / max|row|), max|row| / 127."""
    if x.is_cuda:
        from . import ops

        return ops.quantize_int8(x)
    top = x.detach().double().abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(top)
    codes = torch.round(127 * x.detach().double() / torch.where((top > 0) & ~bad, top, 1.0))
    codes = torch.where(bad, 0.0, codes).to(torch.int8)
    return codes, torch.where(bad, torch.nan, top / 127).float()[..., 0]


class Int8Linear(nn.Module):
    """y = x W^T + b with W and x as 8-bit codes times scales.

    The codes are laid out once, rows of a multiple of 16 bytes, as the kernel
    reads them in place.  Only inference: a call that autograd would record
    raises.  Moving the module moves its buffers; casting it leaves them as
    they are (codes int8, scales and bias float32)."""

    # as a phase-quantized layer: the attention behind a qkv layer runs on the device kernel
    use_packed = True

    def __init__(self, in_features: int, out_features: int, bias: bool = True, device=None):
        super().__init__()
        if in_features < 1 or out_features < 1 or in_features > 131072:
            raise ValueError(f"Int8Linear: {in_features} x {out_features} features (1 .. 131072 in, 1 or more out)")
        self.in_features, self.out_features = in_features, out_features
        self.register_buffer("codes", torch.zeros(out_features, -(-in_features // 16) * 16, dtype=torch.int8, device=device))
        self.register_buffer("weight_scale", torch.zeros(out_features, device=device))
        self.register_buffer("bias", torch.zeros(out_features, device=device) if bias else None)

    @classmethod
    def from_linear(cls, layer: nn.Linear) -> "Int8Linear":
        """The layer's float weight in 8 bits (of a phase-quantized layer: its
        float32 master weight)."""
        if getattr(layer, "_override", None) is not None:
            raise ValueError("Int8Linear.from_linear: the layer runs from supplied codes, not from its float weight")
        weight = layer.weight.detach()
        new = cls(layer.in_features, layer.out_features, layer.bias is not None, weight.device)
        codes, scale = quantize_rows(weight.contiguous())
        new.codes[:, :layer.in_features] = codes
        new.weight_scale.copy_(scale)
        if layer.bias is not None:
            new.bias.copy_(layer.bias.detach())
        return new.train(layer.training)

    def _apply(self, fn, recurse=True):
        return super()._apply(lambda t: t.to(fn(t).device), recurse)

    @property
    def weight_codes(self) -> torch.Tensor:
        return self.codes[:, :self.in_features]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.is_cuda:
            from . import ops

            # the padding is zeros, so rows that fill it are contracted whole
            weight = self.codes if self.codes.shape[1] == self.in_features else self.weight_codes
            return ops.linear_int8(x, weight, self.weight_scale, self.bias)
        if torch.is_grad_enabled() and x.requires_grad:
            raise RuntimeError("Int8Linear has no gradient: call it under torch.no_grad()")
        if x.shape[-1] != self.in_features:
            raise ValueError(f"expected last dim {self.in_features}, got {x.shape[-1]}")
        codes, scale = quantize_rows(x)
        y = (codes.double() @ self.weight_codes.double().t()) * scale[..., None].double() * self.weight_scale.double()
        return (y if self.bias is None else y + self.bias.double()).to(x.dtype)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
