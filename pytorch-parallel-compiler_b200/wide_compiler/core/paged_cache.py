"""WidePagedCache: the paged key-value cache of N fused models.

Pages [N, pages, Hk, page, D] of keys and of values, and a table that names,
for every sequence, the pages its tokens lie in: token p of a sequence is in
page ``table[..., p // page]`` of its model's pool at offset ``p % page``. The
pages hold the model's own type, ``int8`` or ``float8_e4m3fn``; the 8-bit types
keep one fp32 scale per (token, head). The object only holds the tensors: the
caller owns the pool, hands pages out and keeps the lengths. ``ops.cache_write``
and ``ops.qk_norm_rope_write`` fill it, ``ops.cache_read`` reads tokens back and
``ops.decode_attention`` attends over it.
"""
from __future__ import annotations

import struct
from typing import Optional

import torch
from torch import Tensor

from .. import _native as N

_pack = struct.Struct('=5q').pack
CODE_DTYPES = {torch.int8: N.I8, torch.float8_e4m3fn: N.E4M3}


class WidePagedCache:
    __slots__ = ('k', 'v', 'table', 'k_scale', 'v_scale', 'fmt', 'quantized', 'sizes', 'geom')

    def __init__(self, k: Tensor, v: Tensor, table: Tensor, k_scale: Optional[Tensor] = None,
                 v_scale: Optional[Tensor] = None):
        what = "WidePagedCache"
        shape, dtype = k.shape, k.dtype
        if len(shape) != 5 or v.shape != shape or v.dtype != dtype:
            raise ValueError(f"{what}: k and v must be alike, [N, pages, Hk, page, D]; got {tuple(shape)} "
                             f"{dtype} and {tuple(v.shape)} {v.dtype}")
        if not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError(f"{what}: the pages must be contiguous")
        self.fmt = CODE_DTYPES.get(dtype)
        self.quantized = self.fmt is not None
        if self.quantized:
            for s in (k_scale, v_scale):
                if s is None or s.shape != shape[:4] or s.dtype != torch.float32 or not s.is_contiguous():
                    raise ValueError(f"{what}: {dtype} pages need contiguous float32 scales {tuple(shape[:4])}")
        else:
            self.fmt = N.dtype_code(k)
            if k_scale is not None or v_scale is not None:
                raise ValueError(f"{what}: scales belong to int8 and float8_e4m3fn pages, not {dtype}")
        n, pages, kv_heads, page_size, head_dim = shape
        if page_size < 1 and pages > 0:
            raise ValueError(f"{what}: pages of {page_size} tokens")
        ts, st = table.shape, table.stride()
        if table.dtype != torch.int32 or len(ts) not in (2, 3) or (len(ts) == 3 and ts[0] != n) \
                or (ts[-1] > 1 and st[-1] != 1):
            raise ValueError(f"{what}: the table must be int32 [B, M] or [N={n}, B, M] with dense rows, got "
                             f"{tuple(ts)} {table.dtype}")
        self.k, self.v, self.table, self.k_scale, self.v_scale = k, v, table, k_scale, v_scale
        self.sizes = (n, ts[-2], kv_heads, head_dim)              # N, B, Hk, D
        self.geom = _pack(pages, max(page_size, 1), ts[-1], st[0] if len(ts) == 3 else 0, st[-2])

    n = property(lambda self: self.sizes[0])
    batch = property(lambda self: self.sizes[1])
    kv_heads = property(lambda self: self.sizes[2])
    head_dim = property(lambda self: self.sizes[3])
    pages = property(lambda self: self.k.shape[1])
    page_size = property(lambda self: self.k.shape[3])

    @property
    def max_len(self) -> int:
        """Tokens that one sequence's table row spans."""
        return self.table.shape[-1] * self.page_size

    @classmethod
    def allocate(cls, n: int, batch: int, kv_heads: int, head_dim: int, max_len: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device='cuda') -> 'WidePagedCache':
        """A cache with room for ``max_len`` tokens of every sequence, its
        pages handed out in order (one table for all models)."""
        if page_size < 1 or max_len < 0:
            raise ValueError(f"WidePagedCache: pages of {page_size} tokens for {max_len}")
        cols = -(-max_len // page_size)
        shape = (n, batch * cols, kv_heads, page_size, head_dim)
        k, v = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
        table = torch.arange(batch * cols, dtype=torch.int32, device=device).view(batch, cols)
        if dtype not in CODE_DTYPES:
            return cls(k, v, table)
        scale = lambda: torch.empty(shape[:4], dtype=torch.float32, device=device)
        return cls(k, v, table, scale(), scale())

    def __repr__(self):
        return (f"WidePagedCache({self.n}x[{self.pages} pages of {self.page_size}, heads={self.kv_heads}, "
                f"d={self.head_dim}], {self.k.dtype}, {self.batch} sequences of up to {self.max_len})")


__all__ = ['WidePagedCache']
