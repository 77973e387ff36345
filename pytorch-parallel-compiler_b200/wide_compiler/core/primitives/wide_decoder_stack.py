"""WideDecoderStack: the layers of N decoders, their norms fused into the
residual stream.

A layer is attention and a feed-forward block (two linear layers with a GELU
between them) on one residual stream x. What stands between two blocks is one
operator (``ops.residual_norm``): the last block's output y is normed (where
there are post norms), gated, scaled and added to x, and the sum is normed for
the next block,

    x <- x + residual_scale * gate * post(y),   z = norm(x)

The first block's norm reads the stream alone, and the last sum is normed for
the caller. Parameters are N-first: ``WideDecoderAttention`` and ``WideLinear``
modules, norm weights (and LayerNorm biases) [N, d_model], learned gates
[N, d_model].

``quantize_()`` makes the served form: 8-bit projections and linear layers, the
norms straight into their codes (``ops.residual_norm_quantize``).
"""
from __future__ import annotations

from typing import Callable, List, Optional, Sequence

import torch
from torch import Tensor, nn

from ... import ops
from ..paged_cache import WidePagedCache
from .wide_decoder_attention import WideDecoderAttention
from .wide_linear import WideLinear
from .wide_linear_int8 import WideLinearInt8


class _Norm(nn.Module):
    """Weight and, for a LayerNorm, bias of one norm of N models."""

    def __init__(self, n: int, d: int, center: bool):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(n, d))
        self.register_parameter('bias', nn.Parameter(torch.zeros(n, d)) if center else None)


class WideDecoderLayer(nn.Module):
    """The parameters of one layer; WideDecoderStack runs it."""

    def __init__(self, n: int, d_model: int, hidden: int, attn: WideDecoderAttention, center: bool, post_norm: bool,
                 gate_init: Optional[float], bias: bool):
        super().__init__()
        self.attn = attn
        self.up, self.down = WideLinear(n, d_model, hidden, bias), WideLinear(n, hidden, d_model, bias)
        for block in ('attn', 'mlp'):
            self.add_module(block + '_norm', _Norm(n, d_model, center))
            self.add_module(block + '_post', _Norm(n, d_model, center) if post_norm else None)
            self.register_parameter(block + '_gate', None if gate_init is None else
                                    nn.Parameter(torch.full((n, d_model), float(gate_init))))

    def mlp(self, z) -> Tensor:
        if isinstance(self.up, WideLinearInt8):
            return self.down(self.up(z, ops.ACT_GELU))
        return self.down(ops.linear(z, self.up.weight, self.up.bias, ops.ACT_GELU))


class WideDecoderStack(nn.Module):
    def __init__(self, n: int, d_model: int, layers: int, n_heads: int, n_kv_heads: Optional[int] = None,
                 hidden: Optional[int] = None, norm: str = 'rms', post_norm: bool = False,
                 gate_init: Optional[float] = None, residual_scale: float = 1.0, eps: float = 1e-6, bias: bool = False,
                 **attention):
        """``norm``: 'rms' or 'layer'; ``post_norm``: each block's output is normed
        as well; ``gate_init``: learned gates [N, d_model] that start there;
        ``attention``: further arguments of WideDecoderAttention (head_dim,
        rotary_dim, max_positions, theta, interleaved)."""
        super().__init__()
        if norm not in ('rms', 'layer'):
            raise ValueError(f"WideDecoderStack: norm must be 'rms' or 'layer', got {norm!r}")
        self.n, self.d_model, self.center = n, d_model, norm == 'layer'
        self.residual_scale, self.eps, self.quantized = residual_scale, eps, False
        hidden = 4 * d_model if hidden is None else hidden
        self.layers = nn.ModuleList(
            WideDecoderLayer(n, d_model, hidden, WideDecoderAttention(n, d_model, n_heads, n_kv_heads, bias=bias,
                                                                      **attention),
                             self.center, post_norm, gate_init, bias) for _ in range(layers))
        self.norm = _Norm(n, d_model, self.center)

    @torch.no_grad()
    def quantize_(self) -> 'WideDecoderStack':
        """Turns all linear layers (on the GPU) into 8-bit ones, in place, for
        serving: there is no gradient from then on. Goes layer by layer; after a
        failure (no memory) the rest is as it was, and a next call goes on there."""
        if not self.quantized:
            for layer in self.layers:
                up, down = (m if isinstance(m, WideLinearInt8) else WideLinearInt8.from_wide(m)
                            for m in (layer.up, layer.down))
                layer.attn.quantize_()
                layer.up, layer.down = up, down
            self.quantized = True
            self.requires_grad_(False)
        return self

    def _boundary(self, x: Tensor, y: Optional[Tensor], norm: _Norm, edge, quantize: bool):
        post, gate = edge
        args = (x, y, norm.weight, norm.bias, None if post is None else post.weight, None if post is None else post.bias,
                gate, self.residual_scale, self.eps, self.center)
        if quantize:
            x, codes, scales = ops.residual_norm_quantize(*args)
            return x, (codes, scales)
        return ops.residual_norm(*args)

    def _run(self, x: Tensor, attend: Callable, gates: Optional[Sequence[Tensor]]) -> Tensor:
        if x.dim() != 4 or x.shape[0] != self.n or x.shape[3] != self.d_model:
            raise ValueError(f"WideDecoderStack: input must be [N={self.n}, B, T, D={self.d_model}], got "
                             f"{tuple(x.shape)}")
        if gates is not None and len(gates) != 2 * len(self.layers):
            raise ValueError(f"WideDecoderStack: {len(gates)} gates for {len(self.layers)} layers of two blocks")
        y, edge = None, (None, None)
        for i, layer in enumerate(self.layers):
            of = (layer.attn_gate, layer.mlp_gate) if gates is None else gates[2 * i:2 * i + 2]
            x, z = self._boundary(x, y, layer.attn_norm, edge, self.quantized)
            y, edge = attend(i, layer.attn, z), (layer.attn_post, of[0])
            x, z = self._boundary(x, y, layer.mlp_norm, edge, self.quantized)
            y, edge = layer.mlp(z), (layer.mlp_post, of[1])
        return self._boundary(x, y, self.norm, edge, False)[1]

    def new_caches(self, batch: int, max_len: int, page_size: int = 64, dtype: Optional[torch.dtype] = None
                   ) -> List[WidePagedCache]:
        """A cache for each layer."""
        return [layer.attn.new_cache(batch, max_len, page_size, dtype) for layer in self.layers]

    def forward(self, x: Tensor, positions: Optional[Tensor] = None, gates: Optional[Sequence[Tensor]] = None) -> Tensor:
        """x [N, B, T, d_model] -> the normed stream after the last layer, causal
        over T (differentiable until it is quantised). ``gates``: one for each
        block ([N, D], [N, B, D] or [N, B, T, D]) instead of the learned ones."""
        return self._run(x, lambda i, attn, z: attn(z, positions), gates)

    @torch.no_grad()
    def prefill(self, x: Tensor, caches: Sequence[WidePagedCache], positions: Optional[Tensor] = None,
                gates: Optional[Sequence[Tensor]] = None) -> Tensor:
        """``forward`` on prompts, whose keys and values go to the caches."""
        return self._run(x, lambda i, attn, z: attn.prefill(z, caches[i], positions), gates)

    @torch.no_grad()
    def step(self, x: Tensor, caches: Sequence[WidePagedCache], lengths: Tensor, window: int = 0,
             gates: Optional[Sequence[Tensor]] = None) -> Tensor:
        """One new token of every sequence: x [N, B, 1, d_model], ``lengths`` [B] or
        [N, B] with it (see WideDecoderAttention.step)."""
        return self._run(x, lambda i, attn, z: attn.step(z, caches[i], lengths, window), gates)

    def __repr__(self):
        kind = 'layer' if self.center else 'rms'
        return (f"WideDecoderStack({self.n}x[d={self.d_model}, layers={len(self.layers)}, norm={kind}"
                f"{', int8' if self.quantized else ''}])")


__all__ = ['WideDecoderStack', 'WideDecoderLayer']
