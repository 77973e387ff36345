"""Generating with N fused language models.

N small decoders (token embedding, layers of LayerNorm -> WideDecoderAttention
-> LayerNorm -> two Linear layers, a vocabulary projection) run as one wide
model: each continues its own prompts, greedily, over a paged key-value cache.
The prompt goes through ``prefill`` once, then every token is one ``step``.
With ``--stack`` the layers are a WideDecoderStack (norms fused into the residual
stream), with ``--int8`` its linear layers run on 8-bit weights.

    python examples/wide_decoder.py [--models 8] [--batch 4] [--prompt 64] [--new 32] [--cache int8] [--stack] [--int8]
"""
from __future__ import annotations

import argparse
import os
import sys
import time

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "pytorch-parallel-compiler_b200"))

import torch  # noqa: E402
from torch import Tensor, nn  # noqa: E402

import wide_compiler as wc  # noqa: E402
from wide_compiler import ops  # noqa: E402


class WideDecoder(nn.Module):
    def __init__(self, n: int, vocab: int, d_model: int, layers: int, heads: int, kv_heads: int, max_len: int):
        super().__init__()
        self.n, self.vocab, self.max_len = n, vocab, max_len
        self.embed = nn.Parameter(torch.randn(n, vocab, d_model) * 0.5)
        self.layers = nn.ModuleList()
        for _ in range(layers):
            self.layers.append(nn.ModuleDict(dict(
                norm1=wc.WideLayerNorm(n, d_model),
                attn=wc.WideDecoderAttention(n, d_model, heads, kv_heads, max_positions=max_len),
                norm2=wc.WideLayerNorm(n, d_model),
                up=wc.WideLinear(n, d_model, 4 * d_model),
                down=wc.WideLinear(n, 4 * d_model, d_model))))
        self.norm = wc.WideLayerNorm(n, d_model)
        self.head = wc.WideLinear(n, d_model, vocab)

    def caches(self, batch: int, page_size: int = 16, dtype=None):
        return [layer['attn'].new_cache(batch, self.max_len, page_size, dtype) for layer in self.layers]

    def _tokens(self, tokens: Tensor) -> Tensor:
        """[N, B, T] token ids -> [N, B, T, d_model]: each model its own rows."""
        n = torch.arange(self.n, device=tokens.device)[:, None, None]
        return self.embed[n, tokens]

    def _run(self, tokens: Tensor, attend) -> Tensor:
        x = self._tokens(tokens)
        for i, layer in enumerate(self.layers):
            x = ops.binary(x, attend(i, layer['attn'], layer['norm1'](x)), 'add')
            x = ops.binary(x, layer['down'](ops.unary(layer['up'](layer['norm2'](x)), 'gelu')), 'add')
        return self.head(self.norm(x))

    def forward(self, tokens: Tensor) -> Tensor:
        """Logits [N, B, T, vocab] of whole sequences (differentiable)."""
        return self._run(tokens, lambda i, attn, x: attn(x))

    def prefill(self, tokens: Tensor, caches, positions: Tensor) -> Tensor:
        return self._run(tokens, lambda i, attn, x: attn.prefill(x, caches[i], positions))

    def step(self, tokens: Tensor, caches, lengths: Tensor) -> Tensor:
        return self._run(tokens, lambda i, attn, x: attn.step(x, caches[i], lengths))

    @torch.no_grad()
    def generate(self, prompts: Tensor, prompt_lengths: Tensor, new: int, cache_dtype=None):
        """prompts [N, B, T] (padded at the end), prompt_lengths [N, B]. Returns
        the new tokens [N, B, new] and the logits they were taken from. (A
        prompt of no tokens goes on from its first padded one.)"""
        n, b, t = prompts.shape
        if t + new - 1 > self.max_len:
            raise ValueError(f"prompts of {t} tokens and {new} more go past max_len = {self.max_len}")
        caches = self.caches(b, dtype=cache_dtype)
        pos = torch.arange(t, device=prompts.device).expand(n, b, t)
        pos = torch.where(pos < prompt_lengths[..., None], pos, torch.full_like(pos, -1))
        logits = self.prefill(prompts, caches, pos)
        last = (prompt_lengths - 1).clamp(min=0).long()[..., None, None].expand(n, b, 1, self.vocab)
        logits = logits.gather(2, last)
        out, lengths, kept = [], prompt_lengths.clone(), []
        for i in range(new):
            kept.append(logits)
            out.append(logits.argmax(-1))
            if i + 1 < new:
                lengths = lengths + 1
                logits = self.step(out[-1], caches, lengths)
        return torch.cat(out, -1), torch.cat(kept, 2)


class WideStackDecoder(WideDecoder):
    """The same decoder with a WideDecoderStack for its layers and last norm."""

    def __init__(self, n: int, vocab: int, d_model: int, layers: int, heads: int, kv_heads: int, max_len: int):
        super().__init__(n, vocab, d_model, 0, heads, kv_heads, max_len)
        self.stack = wc.WideDecoderStack(n, d_model, layers, heads, kv_heads, post_norm=True, max_positions=max_len)
        self.norm = nn.Identity()                        # the stack's last norm

    def caches(self, batch: int, page_size: int = 16, dtype=None):
        return self.stack.new_caches(batch, self.max_len, page_size, dtype)

    def forward(self, tokens: Tensor) -> Tensor:
        return self.head(self.stack(self._tokens(tokens)))

    def prefill(self, tokens: Tensor, caches, positions: Tensor) -> Tensor:
        return self.head(self.stack.prefill(self._tokens(tokens), caches, positions))

    def step(self, tokens: Tensor, caches, lengths: Tensor) -> Tensor:
        return self.head(self.stack.step(self._tokens(tokens), caches, lengths))


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--models", type=int, default=8)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=64)
    ap.add_argument("--new", type=int, default=32)
    ap.add_argument("--cache", choices=("model", "int8", "fp8"), default="model")
    ap.add_argument("--stack", action="store_true")
    ap.add_argument("--int8", action="store_true")
    a = ap.parse_args()
    torch.manual_seed(0)
    kind = WideStackDecoder if a.stack or a.int8 else WideDecoder
    model = kind(a.models, 1000, 512, 2, 8, 2, a.prompt + a.new).to("cuda", torch.bfloat16).eval()
    if a.int8:
        model.stack.quantize_()
    prompts = torch.randint(0, 1000, (a.models, a.batch, a.prompt), device="cuda")
    lengths = torch.randint(a.prompt // 2, a.prompt + 1, (a.models, a.batch), device="cuda", dtype=torch.int32)
    dtype = {"model": None, "int8": torch.int8, "fp8": torch.float8_e4m3fn}[a.cache]
    for _ in range(2):
        torch.cuda.synchronize()
        t = time.perf_counter()
        tokens, _ = model.generate(prompts, lengths, a.new, dtype)
        torch.cuda.synchronize()
        t = time.perf_counter() - t
    print(f"{a.models} models x {a.batch} sequences x {a.new} tokens in {t * 1e3:.1f} ms "
          f"({a.models * a.batch * a.new / t:.0f} tokens/s)")
    print("first model, first sequence:", tokens[0, 0].tolist())


if __name__ == "__main__":
    main()
