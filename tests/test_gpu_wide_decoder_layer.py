"""GPU tests of WideDecoderAttention and the example that generates with it:
the prompt and step paths against the whole-sequence path, the gradients
against the torch formulation."""
import os
import sys

import pytest
import torch

import decoder_ref as R
import wide_compiler as wc
from conftest import ROOT
from gpu_util import FP32_TOL, assert_lowp_close, no_device_error
from wide_compiler import _autograd as AG
from wide_compiler import ops

sys.path.insert(0, os.path.join(ROOT, "examples"))
from wide_decoder import WideDecoder  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def close(got, want, dtype):
    if dtype == torch.float32:
        torch.testing.assert_close(got, want, **FP32_TOL)
    else:
        assert_lowp_close(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [dict(n_kv_heads=2), dict(rotary_dim=16, interleaved=True, bias=True),
                                dict(n_kv_heads=1, head_dim=48, rotary_dim=24)])
def test_prompt_then_steps_equal_the_whole_sequence(dtype, kw):
    torch.manual_seed(0)
    n, b, t, prompt, d = 3, 2, 21, 9, 128
    layer = wc.WideDecoderAttention(n, d, 4, max_positions=64, **kw).to(DEV, dtype)
    with torch.no_grad():
        for p in (layer.q_norm, layer.k_norm):
            p.copy_(1 + 0.2 * torch.randn_like(p))
    x = torch.randn(n, b, t, d, device=DEV).to(dtype)
    whole = layer(x)
    cache = layer.new_cache(b, t, page_size=4)
    close(layer.prefill(x[:, :, :prompt], cache), whole[:, :, :prompt], dtype)
    lengths = torch.full((b,), prompt, device=DEV, dtype=torch.int32)
    for i in range(prompt, t):
        lengths = lengths + 1
        close(layer.step(x[:, :, i:i + 1], cache, lengths), whole[:, :, i:i + 1], dtype)
    no_device_error()


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn])
def test_steps_over_a_quantised_cache_follow_its_values(fmt):
    """A step over 8-bit pages is attention over the values they hold."""
    torch.manual_seed(1)
    n, b, t, d = 2, 3, 17, 64
    layer = wc.WideDecoderAttention(n, d, 4, 2, max_positions=64).to(DEV, torch.bfloat16)
    x = torch.randn(n, b, t, d, device=DEV).to(torch.bfloat16)
    cache = layer.new_cache(b, t, page_size=8, dtype=fmt)
    layer.prefill(x[:, :, :t - 1], cache)
    lengths = torch.full((b,), t, device=DEV, dtype=torch.int32)
    out = layer.step(x[:, :, t - 1:], cache, lengths)
    q, k, v = layer._project(x[:, :, t - 1:])
    q, _ = ops.qk_norm_rope(q, k, layer.q_norm, layer.k_norm, *layer.rotation(x.device), (lengths - 1).unsqueeze(-1))
    o, _, _ = R.decode(q[:, :, 0], cache, lengths)
    want = torch.einsum('nod,nbd->nbo', layer.out_weight.double().cpu(), o.flatten(-2))
    assert_lowp_close(out[:, :, 0], want)


def test_ragged_prompts_and_left_out_sequences():
    torch.manual_seed(2)
    n, b, t, d = 2, 3, 8, 64
    layer = wc.WideDecoderAttention(n, d, 4, 2, max_positions=64).to(DEV)
    x = torch.randn(n, b, t + 1, d, device=DEV)
    keep = torch.tensor([[8, 3, 0], [1, 8, 5]], device=DEV, dtype=torch.int32)
    pos = torch.arange(t, device=DEV).expand(n, b, t)
    pos = torch.where(pos < keep[..., None], pos, torch.full_like(pos, -1))
    cache = layer.new_cache(b, t + 1, page_size=4)
    layer.prefill(x[:, :, :t], cache, pos)
    lengths = torch.where(keep > 0, keep + 1, torch.zeros_like(keep))
    out = layer.step(x[:, :, t:], cache, lengths)
    for i in range(n):
        for j in range(b):
            m = int(keep[i, j])
            if m == 0:
                assert float(out[i, j].abs().max()) == 0.0
                continue
            seq = torch.cat([x[:, j:j + 1, :m], x[:, j:j + 1, t:]], 2)
            torch.testing.assert_close(out[i, j, 0], layer(seq)[i, 0, -1], **FP32_TOL)
    no_device_error()


@pytest.mark.grad
@pytest.mark.parametrize("kv_heads", [1, 2, 4])
def test_layer_gradients(kv_heads):
    torch.manual_seed(3)
    n, b, t, d = 2, 2, 7, 64
    layer = wc.WideDecoderAttention(n, d, 4, kv_heads, rotary_dim=8, max_positions=16, bias=True).to(DEV)
    x = torch.randn(n, b, t, d, device=DEV, requires_grad=True)
    dy = torch.randn(n, b, t, d, device=DEV)
    got = torch.autograd.grad(layer(x), [x, *layer.parameters()], dy)

    def plain(x):
        qkv = AG.linear_t(x, layer.qkv_weight, layer.qkv_bias)
        hd = layer.head_dim
        cut = lambda a, h: qkv[..., a * hd:(a + h) * hd].unflatten(-1, (h, hd))
        q, k, v = cut(0, 4), cut(4, kv_heads), cut(4 + kv_heads, kv_heads)
        q, k = AG.qk_norm_rope_t(q, k, layer.q_norm, layer.k_norm, *layer.rotation(x.device),
                                 torch.arange(t, device=DEV), layer.eps, False)
        return AG.linear_t(AG.causal_attention_t(q, k, v).flatten(-2), layer.out_weight, layer.out_bias)

    want = torch.autograd.grad(plain(x), [x, *layer.parameters()], dy)
    for g, w in zip(got, want):
        torch.testing.assert_close(g, w, **FP32_TOL)


@pytest.mark.parametrize("cache_dtype", [None, torch.int8, torch.float8_e4m3fn])
def test_example_generates_what_whole_sequences_score(cache_dtype):
    """Every step's logits against one pass over the finished sequences: the
    fp32 model exactly, 8-bit caches within what their rounding moves."""
    torch.manual_seed(4)
    n, b, t, new = 3, 2, 11, 6
    model = WideDecoder(n, 50, 64, 2, 4, 2, t + new).to(DEV).eval()
    prompts = torch.randint(0, 50, (n, b, t), device=DEV)
    lengths = torch.tensor([[11, 4], [7, 11], [1, 9]], device=DEV, dtype=torch.int32)
    tokens, logits = model.generate(prompts, lengths, new, cache_dtype)
    assert tokens.shape == (n, b, new) and torch.equal(tokens, logits.argmax(-1))
    for i in range(n):
        for j in range(b):
            m = int(lengths[i, j])
            seq = torch.cat([prompts[:, j:j + 1, :m], tokens[:, j:j + 1, :-1]], 2)
            want = model(seq)[i, 0, m - 1:]
            if cache_dtype is None:
                torch.testing.assert_close(logits[i, j], want, **FP32_TOL)
            else:
                assert_lowp_close(logits[i, j], want, rtol=0.0, atol_frac=0.15)
    no_device_error()


def test_decode_step_in_a_cuda_graph():
    """A whole layer's step recorded once and replayed with new tokens."""
    torch.manual_seed(6)
    n, b, d = 2, 3, 64
    layer = wc.WideDecoderAttention(n, d, 4, 2, max_positions=64).to(DEV, torch.bfloat16)
    cache, ref = layer.new_cache(b, 32, page_size=8), layer.new_cache(b, 32, page_size=8)
    prompt = torch.randn(n, b, 5, d, device=DEV).to(torch.bfloat16)
    for c in (cache, ref):
        layer.prefill(prompt, c)
    x = torch.randn(n, b, 1, d, device=DEV).to(torch.bfloat16)
    lengths = torch.full((b,), 6, device=DEV, dtype=torch.int32)
    scratch = layer.new_cache(b, 32, page_size=8)
    layer.step(x, scratch, lengths)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layer.step(x, cache, lengths)
    for i in range(3):
        x.copy_(torch.randn_like(x))
        lengths.fill_(6 + i)
        g.replay()
        assert torch.equal(out, layer.step(x, ref, lengths))
