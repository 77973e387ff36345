"""WideLinearInt8: N linear layers served with 8-bit weights.

Weights are int8 codes with one fp32 scale for each output channel, the rows of
the input are quantised as they come (one scale a token), and the products are
summed in int32 (``ops.quantize_rows``, ``ops.linear_int8``). Made from trained
WideLinear layers; there is no gradient.

Buffers: ``weight`` int8 [N, out, in rounded up to 16] (zeros past ``in``),
``weight_scale`` float32 [N, out], which stays float32 when the module is cast,
``bias`` [N, out] in the type of the results, or None.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor, nn

from ... import ops
from .wide_linear import WideLinear


class WideLinearInt8(nn.Module):
    def __init__(self, n: int, in_features: int, out_features: int, bias: bool = True,
                 dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        self.n, self.in_features, self.out_features, self.dtype = n, in_features, out_features, dtype
        width = -(-in_features // 16) * 16
        self.register_buffer('weight', torch.zeros(n, out_features, width, dtype=torch.int8, device=device))
        self.register_buffer('weight_scale', torch.ones(n, out_features, dtype=torch.float32, device=device))
        self.register_buffer('bias', torch.zeros(n, out_features, dtype=dtype, device=device) if bias else None)

    def _apply(self, fn, recurse=True):
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != torch.float32:             # a cast of the module: scales keep their bits
            self.weight_scale = scale.to(device=self.weight_scale.device)
        self.dtype = fn(torch.empty(0, dtype=self.dtype, device=scale.device)).dtype
        return self

    @property
    def codes(self) -> Tensor:
        """The weights' codes [N, out, in], rows 16 bytes (or a multiple) apart."""
        return self.weight[..., :self.in_features]

    @torch.no_grad()
    def load_weight(self, weight: Tensor, bias: Optional[Tensor] = None) -> 'WideLinearInt8':
        """Quantises weight [N, out, in] (on the GPU) into this layer."""
        if weight.shape != (self.n, self.out_features, self.in_features) or (bias is None) != (self.bias is None):
            raise ValueError(f"{self!r}: weight {tuple(weight.shape)}, bias {None if bias is None else tuple(bias.shape)}")
        codes, scale = ops.quantize_rows(weight)
        self.codes.copy_(codes)
        self.weight_scale.copy_(scale)
        if bias is not None:
            self.bias.copy_(bias)
        return self

    @classmethod
    def from_weight(cls, weight: Tensor, bias: Optional[Tensor] = None) -> 'WideLinearInt8':
        n, o, k = weight.shape
        return cls(n, k, o, bias is not None, weight.dtype, weight.device).load_weight(weight.detach(), bias)

    @classmethod
    def from_wide(cls, linear: WideLinear) -> 'WideLinearInt8':
        """The 8-bit form of a trained layer (on the GPU)."""
        return cls.from_weight(linear.weight, linear.bias)

    def forward(self, x: Union[Tensor, Tuple[Tensor, Tensor]], act: int = ops.ACT_NONE) -> Tensor:
        """x [N, ..., in], or its (codes, scales); -> [N, ..., out] with the
        activation ``act``."""
        codes, scale = x if isinstance(x, tuple) else ops.quantize_rows(x)
        return ops.linear_int8(codes, scale, self.codes, self.weight_scale, self.bias, act, self.dtype)

    def __repr__(self):
        return f"WideLinearInt8({self.n}x[{self.in_features}->{self.out_features}])"


__all__ = ['WideLinearInt8']
