"""WideDecoderAttention: N causal self-attention layers that can generate.

What WideAttention lacks for decoding: grouped key heads, an RMS norm of every
query and key head with the position rotation, and a paged key-value cache.
Three ways through one set of parameters:

  forward   a whole sequence, differentiable (training, scoring)
  prefill   a prompt: the same result, its keys and values written to a cache
  step      one new token for every sequence, attending over the cache

Parameters are N-first: ``qkv_weight`` [N, (Hq + 2 Hk) D, d_model] (queries,
then keys, then values), ``q_norm`` / ``k_norm`` [N, D], ``out_weight``
[N, d_model, Hq D], optional ``qkv_bias`` / ``out_bias``.

Kernels: the projections are grouped GEMMs; norm and rotation run in one pass
over the projection's output in place (``ops.qk_norm_rope``), in a step
together with the cache write (``ops.qk_norm_rope_write``); whole sequences use
the flash-style core, steps ``ops.decode_attention``.
"""
from __future__ import annotations

from typing import List, Optional

import torch
from torch import Tensor, nn

from ... import ops
from ..paged_cache import WidePagedCache


class WideDecoderAttention(nn.Module):
    def __init__(self, n: int, d_model: int, n_heads: int, n_kv_heads: Optional[int] = None,
                 head_dim: Optional[int] = None, rotary_dim: Optional[int] = None, max_positions: int = 4096,
                 theta: float = 10000.0, interleaved: bool = False, eps: float = 1e-6, bias: bool = False):
        super().__init__()
        n_kv_heads = n_heads if n_kv_heads is None else n_kv_heads
        if n_heads % n_kv_heads != 0:
            raise ValueError(f"WideDecoderAttention: {n_heads} query heads over {n_kv_heads} key heads")
        if head_dim is None and d_model % n_heads != 0:
            raise ValueError(f"WideDecoderAttention: d_model ({d_model}) must be divisible by n_heads ({n_heads})")
        self.n, self.d_model, self.n_heads, self.n_kv_heads = n, d_model, n_heads, n_kv_heads
        self.head_dim = d_model // n_heads if head_dim is None else head_dim
        self.rotary_dim = self.head_dim // 2 * 2 if rotary_dim is None else rotary_dim
        self.max_positions, self.theta, self.interleaved, self.eps = max_positions, theta, interleaved, eps
        d, rows = self.head_dim, (n_heads + 2 * n_kv_heads) * self.head_dim
        self.qkv_weight = nn.Parameter(torch.empty(n, rows, d_model))
        self.out_weight = nn.Parameter(torch.empty(n, d_model, n_heads * d))
        self.q_norm = nn.Parameter(torch.ones(n, d))
        self.k_norm = nn.Parameter(torch.ones(n, d))
        for name, width in (('qkv_bias', rows), ('out_bias', d_model)):
            self.register_parameter(name, nn.Parameter(torch.zeros(n, width)) if bias else None)
        for i in range(n):
            nn.init.xavier_uniform_(self.qkv_weight[i])
            nn.init.xavier_uniform_(self.out_weight[i])
        self._tables = {}                # fp32 whatever the module's type, so not buffers

    def rotation(self, device: torch.device, rows: Optional[int] = None):
        """cos / sin [rows, rotary_dim / 2] in fp32 (rows: max_positions unless
        given), angles in 64 bits; made once for each use they serve."""
        key = (device, self.max_positions if rows is None else rows, self.rotary_dim, self.theta)
        if torch.compiler.is_compiling():                # the traced graph makes them
            if key not in self._tables:
                self._tables[key] = self._make_rotation(device, key[1])
            return self._tables[key]
        if key not in self._tables or self._tables[key][0].is_inference():
            if device.type == 'cuda' and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("WideDecoderAttention: the rotation tables cannot be made while a CUDA graph is "
                                   "captured: run the layer once before")
            with torch.inference_mode(False):            # they serve training as well
                self._tables[key] = self._make_rotation(device, key[1])
        return self._tables[key]

    def _make_rotation(self, device: torch.device, rows: int):
        i = torch.arange(0, self.rotary_dim, 2, dtype=torch.float64) / max(self.rotary_dim, 1)
        ang = torch.arange(rows, dtype=torch.float64)[:, None] * self.theta ** -i[None]
        return torch.cos(ang).float().to(device), torch.sin(ang).float().to(device)

    def _cache_rotation(self, x: Tensor, cache: WidePagedCache):
        """Tables that reach as far as the cache (whole pages, or one that the
        caller made): every key that a step's attention sees was written."""
        return self.rotation(x.device, max(self.max_positions, cache.max_len))

    def _positions(self, x: Tensor, positions: Optional[Tensor], most: int) -> Tensor:
        """Positions of x's tokens: those given, or 0, 1, .. below ``most``."""
        if positions is not None:
            return positions
        if x.shape[2] > most:
            raise ValueError(f"WideDecoderAttention: {x.shape[2]} tokens where there are positions for {most}")
        return torch.arange(x.shape[2], device=x.device)

    def _check(self, x: Tensor) -> None:
        if x.dim() != 4 or x.shape[0] != self.n or x.shape[3] != self.d_model:
            raise ValueError(f"WideDecoderAttention: input must be [N={self.n}, B, T, D={self.d_model}], got "
                             f"{tuple(x.shape)}")

    def _project(self, x: Tensor):
        self._check(x)
        qkv = ops.linear(x, self.qkv_weight, self.qkv_bias)
        d, hq, hk = self.head_dim, self.n_heads, self.n_kv_heads
        cut = lambda a, h: qkv[..., a * d:(a + h) * d].unflatten(-1, (h, d))
        return cut(0, hq), cut(hq, hk), cut(hq + hk, hk)

    def _output(self, o: Tensor) -> Tensor:
        return ops.linear(o.flatten(-2), self.out_weight, self.out_bias)

    def new_cache(self, batch: int, max_len: int, page_size: int = 64, dtype: Optional[torch.dtype] = None
                  ) -> WidePagedCache:
        """A cache for this layer; ``dtype`` int8 or float8_e4m3fn quantises it."""
        if max_len > self.max_positions:
            raise ValueError(f"WideDecoderAttention: a cache of {max_len} tokens goes past max_positions = "
                             f"{self.max_positions}")
        return WidePagedCache.allocate(self.n, batch, self.n_kv_heads, self.head_dim, max_len, page_size,
                                       self.qkv_weight.dtype if dtype is None else dtype, self.qkv_weight.device)

    def forward(self, x: Tensor, positions: Optional[Tensor] = None) -> Tensor:
        """x [N, B, T, d_model] -> the same shape, causal over the T tokens
        (padding, whose ``positions`` are negative, at their end)."""
        self._check(x)
        positions = self._positions(x, positions, self.max_positions)
        q, k, v = self._project(x)
        q, k = ops.qk_norm_rope(q, k, self.q_norm, self.k_norm, *self.rotation(x.device), positions, self.eps,
                                self.interleaved)
        return self._output(ops.causal_attention(q, k, v))

    @torch.no_grad()
    def prefill(self, x: Tensor, cache: WidePagedCache, positions: Optional[Tensor] = None) -> Tensor:
        """``forward`` on prompts from position 0, padded at the end where
        ``positions`` ([B, T] or [N, B, T]) is negative, with the keys and
        values written to the cache."""
        self._check(x)
        positions = self._positions(x, positions, min(self.max_positions, cache.max_len))
        q, k, v = self._project(x)
        q, k = ops.qk_norm_rope(q, k, self.q_norm, self.k_norm, *self._cache_rotation(x, cache), positions, self.eps,
                                self.interleaved)
        ops.cache_write(cache, k, v, positions)
        return self._output(ops.causal_attention(q, k, v))

    @torch.no_grad()
    def step(self, x: Tensor, cache: WidePagedCache, lengths: Tensor, window: int = 0) -> Tensor:
        """One new token: x [N, B, 1, d_model]; ``lengths`` [B] or [N, B] are
        the tokens of each sequence with the new one, whose position is
        length - 1 (a length of 0 leaves the sequence out: zeros attend)."""
        q, k, v = self._project(x)
        q = ops.qk_norm_rope_write(q, k, v, self.q_norm, self.k_norm, *self._cache_rotation(x, cache),
                                   (lengths - 1).unsqueeze(-1), cache, self.eps, self.interleaved)
        o = ops.decode_attention(q.squeeze(2), cache, lengths, window=window)
        return self._output(o.unsqueeze(2))

    @classmethod
    def from_modules(cls, modules: List['WideDecoderAttention']) -> 'WideDecoderAttention':
        """Fuses layers of the same configuration (each of any n) into one."""
        t = modules[0]
        wide = cls(sum(m.n for m in modules), t.d_model, t.n_heads, t.n_kv_heads, t.head_dim, t.rotary_dim,
                   t.max_positions, t.theta, t.interleaved, t.eps, t.qkv_bias is not None)
        wide = wide.to(device=t.qkv_weight.device, dtype=t.qkv_weight.dtype)
        with torch.no_grad():
            for name, p in wide.named_parameters():
                p.copy_(torch.cat([getattr(m, name) for m in modules]))
        return wide

    def __repr__(self):
        return (f"WideDecoderAttention({self.n}x[d={self.d_model}, h={self.n_heads}/{self.n_kv_heads}x{self.head_dim}, "
                f"rotary={self.rotary_dim}])")


__all__ = ['WideDecoderAttention']
