"""WideDecoderStack and WideLinearInt8 on the GPU: the layers' arithmetic and its
gradients against plain torch, generation against whole sequences, the served
8-bit form, graphs and torch.compile."""
import math
import os
import sys

import pytest
import torch
import torch.nn.functional as F

import wide_compiler as wc
from conftest import ROOT
from gpu_util import FP32_TOL, assert_lowp_close, no_device_error
from wide_compiler import _autograd as AG
from wide_compiler import ops

sys.path.insert(0, os.path.join(ROOT, "examples"))
from wide_decoder import WideStackDecoder  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def stack(n=2, d=64, layers=2, dtype=torch.float32, seed=0, **kw):
    torch.manual_seed(seed)
    s = wc.WideDecoderStack(n, d, layers, 4, 2, hidden=96, max_positions=64, **kw)
    with torch.no_grad():
        for name, p in s.named_parameters():
            if 'norm' in name or 'post' in name:
                p.add_(0.2 * torch.randn_like(p))
    return s.to(DEV, dtype)


def plain(s, x, gates=None):
    """The stack from plain torch formulas (fp32)."""
    def norm(v, m):
        w, b = m.weight[:, None, None], 0 if m.bias is None else m.bias[:, None, None]
        v = v - v.mean(-1, keepdim=True) if s.center else v
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + s.eps) * w + b

    def attend(a, z):
        qkv = AG.linear_t(z, a.qkv_weight, a.qkv_bias)
        d, hq, hk = a.head_dim, a.n_heads, a.n_kv_heads
        cut = lambda i, h: qkv[..., i * d:(i + h) * d].unflatten(-1, (h, d))
        q, k = AG.qk_norm_rope_t(cut(0, hq), cut(hq, hk), a.q_norm, a.k_norm, *a.rotation(z.device),
                                 torch.arange(z.shape[2], device=z.device), a.eps, a.interleaved)
        return AG.linear_t(AG.causal_attention_t(q, k, cut(hq + hk, hk)).flatten(-2), a.out_weight, a.out_bias)

    def add(x, y, post, gate):
        y = y if post is None else norm(y, post)
        if gate is not None:
            y = y * gate.view(gate.shape[:-1] + (1,) * (4 - gate.dim()) + gate.shape[-1:])
        return x + s.residual_scale * y

    for i, layer in enumerate(s.layers):
        g = (layer.attn_gate, layer.mlp_gate) if gates is None else gates[2 * i:2 * i + 2]
        x = add(x, attend(layer.attn, norm(x, layer.attn_norm)), layer.attn_post, g[0])
        z = norm(x, layer.mlp_norm)
        a = F.gelu(AG.linear_t(z, layer.up.weight, layer.up.bias))
        x = add(x, AG.linear_t(a, layer.down.weight, layer.down.bias), layer.mlp_post, g[1])
    return norm(x, s.norm)


KINDS = [dict(), dict(norm='layer', bias=True), dict(post_norm=True, gate_init=0.7), dict(norm='layer', post_norm=True,
                                                                                         residual_scale=0.4)]


@pytest.mark.grad
@pytest.mark.parametrize("kw", KINDS)
def test_forward_and_gradients(kw):
    s = stack(**kw)
    x = torch.randn(2, 3, 7, 64, device=DEV, requires_grad=True)
    y, want = s(x), plain(s, x)
    torch.testing.assert_close(y, want, **FP32_TOL)
    dy = torch.randn_like(y)
    leaves = [x, *s.parameters()]
    for (name, _), a, b in zip([('x', x), *s.named_parameters()], torch.autograd.grad(y, leaves, dy),
                               torch.autograd.grad(want, leaves, dy)):
        torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-4 * float(b.abs().max() + 1), msg=name)
    no_device_error()


@pytest.mark.grad
def test_gates_that_are_given():
    s = stack(gate_init=1.0)
    x = torch.randn(2, 3, 7, 64, device=DEV)
    gates = [torch.rand(*shape, 64, device=DEV, requires_grad=True) for shape in ((2,), (2, 3), (2, 3, 7), (2, 3))]
    y, want = s(x, gates=gates), plain(s, x, gates)
    torch.testing.assert_close(y, want, **FP32_TOL)
    dy = torch.randn_like(y)
    for a, b in zip(torch.autograd.grad(y, gates, dy), torch.autograd.grad(want, gates, dy)):
        torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-4 * float(b.abs().max() + 1))


@pytest.mark.parametrize("kw", KINDS)
def test_steps_continue_prompts(kw):
    s = stack(**kw)
    x = torch.randn(2, 3, 9, 64, device=DEV)
    want = s(x)
    caches = s.new_caches(3, 16, page_size=4)
    lengths = torch.tensor([5, 6, 2], device=DEV, dtype=torch.int32)
    pos = torch.arange(6, device=DEV).expand(3, 6)
    pos = torch.where(pos < lengths[:, None], pos, torch.full_like(pos, -1))
    y = s.prefill(x[:, :, :6], caches, pos)
    for b in range(3):
        m = int(lengths[b])
        torch.testing.assert_close(y[:, b, :m], want[:, b, :m], **FP32_TOL)
    for i in range(3):
        at = (lengths + i).long()
        tok = x[:, torch.arange(3), at].unsqueeze(2)
        y = s.step(tok, caches, (lengths + i + 1).int())
        torch.testing.assert_close(y[:, :, 0], want[:, torch.arange(3), at], **FP32_TOL)
    no_device_error()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", KINDS)
def test_served_in_8_bits(kw, dtype):
    """Codes are within half a step of 1/127 of a row's largest value: the served
    stack stays near the one it was made from, and its steps near its own whole
    sequences (a value at a code's border may fall to either side)."""
    s = stack(dtype=dtype, **kw)
    x = torch.randn(2, 3, 9, 64, device=DEV).to(dtype)
    full = s(x)
    s.quantize_()
    assert s.layers[0].attn.qkv_weight is None and not any(p.requires_grad for p in s.parameters())
    y = s(x)
    off = (y.double() - full.double()).norm() / full.double().norm()
    assert off < 0.05, off
    caches = s.new_caches(3, 16, page_size=4)
    first = s.prefill(x[:, :, :5], caches)
    assert_lowp_close(first, y[:, :, :5], rtol=2e-2, atol_frac=2e-2)
    for t in range(5, 9):
        z = s.step(x[:, :, t:t + 1], caches, torch.full((3,), t + 1, device=DEV, dtype=torch.int32))
        assert_lowp_close(z, y[:, :, t:t + 1], rtol=2e-2, atol_frac=2e-2)
    no_device_error()


def test_linear_int8_layer():
    torch.manual_seed(1)
    wide = wc.WideLinear(3, 70, 33).to(DEV, torch.bfloat16)
    q = wc.WideLinearInt8.from_wide(wide)
    assert q.weight.shape == (3, 33, 80) and not q.weight[..., 70:].any() and q.dtype == torch.bfloat16
    x = torch.randn(3, 4, 2, 70, device=DEV).to(torch.bfloat16)
    y = q(x)
    assert torch.equal(y, q(ops.quantize_rows(x)))
    w = q.codes.double() * q.weight_scale.double()[..., None]
    c, s = ops.quantize_rows(x)
    want = torch.einsum('nbtk,nok->nbto', c.double() * s.double()[..., None], w) + wide.bias.double()[:, None, None]
    assert_lowp_close(y, want)
    assert (w - wide.weight.double()).abs().amax() <= float(q.weight_scale.max()) * 0.5 * (1 + 2 ** -20)
    other = wc.WideLinearInt8(3, 70, 33).to(DEV)
    other.load_state_dict(q.state_dict())
    assert torch.equal(other(x), y)
    half = q.to(torch.float16)
    assert half.weight_scale.dtype == torch.float32 and half(x.half()).dtype == torch.float16
    with pytest.raises(ValueError, match="weight"):
        q.load_weight(wide.weight[:, :3], wide.bias)


def test_served_step_in_a_graph():
    s = stack(dtype=torch.bfloat16, post_norm=True).quantize_()
    caches, ref = s.new_caches(3, 16, page_size=4), s.new_caches(3, 16, page_size=4)
    x = torch.randn(2, 3, 1, 64, device=DEV).to(torch.bfloat16)
    lengths = torch.ones(3, device=DEV, dtype=torch.int32)
    s.step(x, s.new_caches(3, 16, page_size=4), lengths)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = s.step(x, caches, lengths)
    for t in range(4):
        x.normal_()
        lengths.fill_(t + 1)
        graph.replay()
        assert torch.equal(out, s.step(x, ref, lengths))


def test_example_with_a_stack():
    torch.manual_seed(4)
    n, b, t, new = 3, 2, 11, 6
    model = WideStackDecoder(n, 50, 64, 2, 4, 2, t + new).to(DEV).eval()
    prompts = torch.randint(0, 50, (n, b, t), device=DEV)
    lengths = torch.tensor([[11, 4], [7, 11], [1, 9]], device=DEV, dtype=torch.int32)
    tokens, logits = model.generate(prompts, lengths, new)
    for i in range(n):
        for j in range(b):
            m = int(lengths[i, j])
            seq = torch.cat([prompts[:, j:j + 1, :m], tokens[:, j:j + 1, :-1]], 2)
            torch.testing.assert_close(logits[i, j], model(seq)[i, 0, m - 1:], **FP32_TOL)
    model.stack.quantize_()
    tokens, logits = model.generate(prompts, lengths, new, torch.int8)
    assert tokens.shape == (n, b, new) and logits.isfinite().all()
    no_device_error()


@pytest.mark.grad
def test_operators_under_torch_compile():
    torch.manual_seed(5)
    x, y = torch.randn(2, 3, 4, 40, device=DEV), torch.randn(2, 3, 4, 40, device=DEV)
    w, g = 1 + 0.2 * torch.randn(2, 40, device=DEV), torch.rand(2, 3, 40, device=DEV)
    f = torch.compile(lambda x, y, w, g: ops.residual_norm(x, y, w, post_weight=w, gate=g), fullgraph=True, backend="eager")
    leaves = [v.clone().requires_grad_(True) for v in (x, y, w, g)]
    outs, want = f(*leaves), ops.residual_norm(leaves[0], leaves[1], leaves[2], post_weight=leaves[2], gate=leaves[3])
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    d = (torch.randn_like(x), torch.randn_like(x))
    for a, b in zip(torch.autograd.grad(outs, leaves, d), torch.autograd.grad(want, leaves, d)):
        torch.testing.assert_close(a, b, **FP32_TOL)
    f = torch.compile(lambda x, w: ops.residual_norm(x, None, w), fullgraph=True, backend="eager")
    got, want = f(leaves[0], leaves[2]), ops.residual_norm(leaves[0], None, leaves[2])
    assert torch.equal(got[1], want[1])
    for a, b in zip(torch.autograd.grad(got[1], leaves[::2], d[0]), torch.autograd.grad(want[1], leaves[::2], d[0])):
        torch.testing.assert_close(a, b, **FP32_TOL)
    wq, ws = ops.quantize_rows(torch.randn(2, 24, 40, device=DEV))

    def served(x, y, w, wq, ws):
        h, c, s = ops.residual_norm_quantize(x, y, w)
        a = ops.linear_int8(c, s, wq, ws, act=ops.ACT_GELU, dtype=torch.float32)
        _, c2, s2 = ops.residual_norm_quantize(x, None, w)
        return h, a, ops.linear_int8(c2, s2, wq, ws, dtype=torch.bfloat16), *ops.quantize_rows(x)

    with torch.no_grad():
        for a, b in zip(torch.compile(served, fullgraph=True, backend="eager")(x, y, w, wq, ws), served(x, y, w, wq, ws)):
            assert torch.equal(a, b)
