"""GPU tests of the decoder-attention operators and their layer at the edges of
what they take: positions past a table, caches longer than one, gradients of
gradients, first calls in unusual modes."""
import pytest
import torch

import decoder_ref as R
import wide_compiler as wc
from gpu_util import FP32_TOL, no_device_error
from wide_compiler import _native, ops

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
I8, E4M3 = torch.int8, torch.float8_e4m3fn


def heads(n, b, t, hq, hk, d, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(n, b, t, h, d, generator=gen).to(dtype).to(DEV) for h in (hq, hk, hk)]


@pytest.mark.parametrize("dtype,fmt", [(BF16, BF16), (F32, I8), (F16, E4M3)])
def test_fused_write_past_the_rotation_table_writes_neither_side(dtype, fmt):
    """Inside the cache but past cos / sin: as a padding row, for the key, the
    value and their scales."""
    q, k, v = heads(1, 2, 3, 2, 1, 64, dtype, 1)
    w = torch.ones(1, 64, device=DEV, dtype=dtype)
    cos, sin = (x.to(DEV) for x in R.tables(4, 64))
    cache = wc.WidePagedCache.allocate(1, 2, 1, 64, 16, 4, fmt, DEV)
    for x in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if x is not None:
            x.zero_()
    pos = torch.tensor([[0, 4, 3], [15, 1, 2]], device=DEV)
    y = ops.qk_norm_rope_write(q, k, v, w, w, cos, sin, pos, cache)
    assert _native.device_error() == _native.DEV_ERR_INDEX
    kr, vr = ops.cache_read(cache, pos, dtype=dtype if fmt != dtype else None)
    no_device_error()
    past = (pos >= 4)[None]
    for x in (y, kr, vr):
        assert float(x[past].float().abs().max()) == 0.0
        assert float(x[~past].float().abs().amax((-1, -2)).min()) > 0.0
    for s in (cache.k_scale, cache.v_scale):
        if s is not None:
            assert int((s != 0).sum()) == 4


def test_fused_write_past_the_cache_leaves_the_queries():
    """Past the cache but inside cos / sin: nothing is written, and the
    queries, which do not go there, come out as elsewhere."""
    q, k, v = heads(1, 1, 2, 2, 1, 64, BF16, 2)
    w = torch.ones(1, 64, device=DEV, dtype=BF16)
    cos, sin = (x.to(DEV) for x in R.tables(32, 64))
    cache = wc.WidePagedCache.allocate(1, 1, 1, 64, 8, 4, BF16, DEV)
    cache.k.zero_(), cache.v.zero_()
    pos = torch.tensor([9, 31], device=DEV)
    y = ops.qk_norm_rope_write(q, k, v, w, w, cos, sin, pos, cache)
    assert _native.device_error() == _native.DEV_ERR_INDEX
    assert torch.equal(y, ops.qk_norm_rope(q, k, w, w, cos, sin, pos)[0])
    assert float(cache.k.abs().max()) == 0.0 and float(cache.v.abs().max()) == 0.0
    no_device_error()


@pytest.mark.grad
@pytest.mark.parametrize("compiled", [False, True])
def test_gradient_penalty_through_norm_and_rotation(compiled):
    """The kernels' outputs, and gradients of gradients as the torch
    formulation's; first gradients stay the kernel's."""
    from wide_compiler import _autograd as AG
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(2, 2, 5, 3, 64, generator=gen).to(DEV).requires_grad_(True)
    w = (1 + 0.2 * torch.randn(2, 64, generator=gen)).to(DEV).requires_grad_(True)
    cos, sin = (t.to(DEV) for t in R.tables(8, 32))
    pos = torch.tensor([0, 3, -1, 7, 2], device=DEV)
    call = lambda q, k, w: ops.qk_norm_rope(q, k, w, w * 0.5, cos, sin, pos, 1e-6, True)
    if compiled:
        call = torch.compile(call, fullgraph=True, backend="eager")
    plain = lambda q, k, w: AG.qk_norm_rope_t(q, k, w, w * 0.5, cos, sin, pos, 1e-6, True)

    def penalty(f):
        yq, yk = f(x * 1.5, x[..., :1, :], w)
        g, = torch.autograd.grad((yq ** 3).sum() + (yk ** 2).sum(), x, create_graph=True)
        return torch.autograd.grad((g ** 2).sum(), (x, w))

    for got, want in zip(penalty(call), penalty(plain)):
        torch.testing.assert_close(got, want, rtol=1e-3, atol=1e-3 * float(want.abs().max()))
    no_device_error()


@pytest.mark.grad
@pytest.mark.parametrize("act", ['none', 'relu', 'gelu'])
def test_gradient_penalty_through_a_decoder_layer(act):
    """Projections, norm + rotation and attention of WideDecoderAttention, and
    the norm and activation beside it, against their torch formulations."""
    from wide_compiler import _autograd as AG
    torch.manual_seed(5)
    n, b, t, d = 2, 2, 5, 32
    layer = wc.WideDecoderAttention(n, d, 4, 2, max_positions=8, bias=True).to(DEV)
    norm = wc.WideLayerNorm(n, d).to(DEV)
    up = wc.WideLinear(n, d, d).to(DEV)
    x = torch.randn(n, b, t, d, device=DEV, requires_grad=True)
    params = [*layer.parameters(), *norm.parameters(), *up.parameters()]

    def ours(x):
        y = ops.linear(layer(norm(x)), up.weight, up.bias, {'none': 0, 'relu': 1, 'gelu': 2}[act])
        return y if act == 'none' else ops.unary(y, act)

    def plain(x):
        h = AG.layernorm_t(x, norm.weight, norm.bias, n, d, norm.eps)
        qkv = AG.linear_t(h, layer.qkv_weight, layer.qkv_bias)
        cut = lambda a, c: qkv[..., a * 8:(a + c) * 8].unflatten(-1, (c, 8))
        q, k = AG.qk_norm_rope_t(cut(0, 4), cut(4, 2), layer.q_norm, layer.k_norm, *layer.rotation(x.device),
                                 torch.arange(t, device=DEV), layer.eps, False)
        with torch.nn.attention.sdpa_kernel(torch.nn.attention.SDPBackend.MATH):
            h = AG.linear_t(AG.causal_attention_t(q, k, cut(6, 2)).flatten(-2), layer.out_weight, layer.out_bias)
        y = AG.linear_t(h, up.weight, up.bias, {'none': 0, 'relu': 1, 'gelu': 2}[act])
        return y if act == 'none' else AG.act_t(y, {'relu': 1, 'gelu': 2}[act])

    def penalty(f):
        g, = torch.autograd.grad((f(x) ** 2).sum(), x, create_graph=True)
        return torch.autograd.grad((g ** 2).sum(), [x, *params], allow_unused=True)

    for got, want in zip(penalty(ours), penalty(plain)):
        assert (got is None) == (want is None)
        if got is not None:
            torch.testing.assert_close(got, want, rtol=5e-3, atol=2e-3 * float(want.abs().max()) + 1e-6)


@pytest.mark.grad
def test_gradient_penalty_through_batch_and_group_norm_is_refused():
    for f in (lambda x: ops.groupnorm(x, 2, 2, None, None, 1e-5),
              lambda x: ops.batchnorm(x, 2, 4, None, None, None, None, True, False, 0.1, 1e-5)):
        x = torch.randn(2, 3, 4, 5, device=DEV, requires_grad=True)
        g, = torch.autograd.grad((f(x) ** 3).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad((g ** 2).sum(), x)


def test_steps_into_the_last_page_past_max_positions():
    """A cache's pages may reach past max_positions: steps there give what a
    layer with a longer table gives, and read no key that was not written."""
    torch.manual_seed(6)
    n, b, d, page = 2, 2, 64, 16
    short = wc.WideDecoderAttention(n, d, 4, 2, max_positions=17).to(DEV)
    long = wc.WideDecoderAttention(n, d, 4, 2, max_positions=64).to(DEV)
    long.load_state_dict(short.state_dict())
    x = torch.randn(n, b, 20, d, device=DEV)
    caches = [m.new_cache(b, 17, page_size=page) for m in (short, long)]
    for c in caches:
        c.k.fill_(float('nan'))
    for m, c in zip((short, long), caches):
        m.prefill(x[:, :, :16], c)
    for i in range(16, 20):
        ln = torch.full((b,), i + 1, device=DEV, dtype=torch.int32)
        got, want = (m.step(x[:, :, i:i + 1], c, ln) for m, c in zip((short, long), caches))
        assert torch.isfinite(got).all() and torch.equal(got, want)
    no_device_error()


@pytest.mark.grad
def test_training_after_a_first_use_under_inference_mode():
    torch.manual_seed(7)
    layer = wc.WideDecoderAttention(2, 64, 4, 2, max_positions=16).to(DEV)
    x = torch.randn(2, 2, 5, 64, device=DEV)
    with torch.inference_mode():
        cache = layer.new_cache(2, 16, page_size=4)
        layer.prefill(x, cache)
        layer.step(x[:, :, :1], cache, torch.full((2,), 6, device=DEV, dtype=torch.int32))
        want = layer(x)
    y = layer(x)
    assert torch.equal(y, want)
    y.sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in layer.parameters())


@pytest.mark.grad
def test_layer_under_torch_compile():
    torch.manual_seed(8)
    layer = wc.WideDecoderAttention(2, 64, 4, 2, max_positions=16).to(DEV)
    x = torch.randn(2, 2, 5, 64, device=DEV, requires_grad=True)
    want = layer(x)
    got = torch.compile(layer, backend="eager")(x)
    torch.testing.assert_close(got, want, **FP32_TOL)
    dy = torch.randn_like(want)
    for a, b in zip(torch.autograd.grad(got, [x, *layer.parameters()], dy),
                    torch.autograd.grad(want, [x, *layer.parameters()], dy)):
        torch.testing.assert_close(a, b, **FP32_TOL)


@pytest.mark.grad
@pytest.mark.parametrize("first", ["traced", "eager"])
def test_layer_is_one_graph_under_torch_compile(first):
    """forward with gradients, prefill and step, without a break; the rotation
    tables made in the traced call or before it."""
    torch.manual_seed(9)
    n, b, t, d = 2, 2, 5, 64
    layer, ref = (wc.WideDecoderAttention(n, d, 4, 2, max_positions=16).to(DEV) for _ in range(2))
    ref.load_state_dict(layer.state_dict())
    x = torch.randn(n, b, t + 1, d, device=DEV, requires_grad=True)
    if first == "eager":
        layer(x)
    one = lambda f: torch.compile(f, fullgraph=True, backend="eager")
    got, want = one(layer)(x), ref(x)
    torch.testing.assert_close(got, want, **FP32_TOL)
    dy = torch.randn_like(want)
    for g, w in zip(torch.autograd.grad(got, [x, *layer.parameters()], dy),
                    torch.autograd.grad(want, [x, *ref.parameters()], dy)):
        torch.testing.assert_close(g, w, **FP32_TOL)
    caches = [m.new_cache(b, 8, page_size=4) for m in (layer, ref)]
    y = x.detach()
    assert torch.equal(one(layer.prefill)(y[:, :, :t], caches[0]), ref.prefill(y[:, :, :t], caches[1]))
    ln = torch.full((b,), t + 1, device=DEV, dtype=torch.int32)
    assert torch.equal(one(layer.step)(y[:, :, t:], caches[0], ln), ref.step(y[:, :, t:], caches[1], ln))
    assert torch.equal(layer(x), want)
    no_device_error()


def test_step_first_traced_in_one_graph():
    torch.manual_seed(10)
    layer, ref = (wc.WideDecoderAttention(2, 64, 4, 2, max_positions=16).to(DEV) for _ in range(2))
    ref.load_state_dict(layer.state_dict())
    x, ln = torch.randn(2, 2, 1, 64, device=DEV), torch.ones(2, device=DEV, dtype=torch.int32)
    caches = [m.new_cache(2, 8, page_size=4) for m in (layer, ref)]
    step = torch.compile(layer.step, fullgraph=True, backend="eager")
    assert torch.equal(step(x, caches[0], ln), ref.step(x, caches[1], ln))


def test_gradient_entry_without_rows_gives_weight_gradients_of_zero():
    """The C entry, for callers other than ops.qk_norm_rope_bwd."""
    import struct
    n, b, t, hq, hk, d = 2, 3, 0, 4, 2, 64
    geom = struct.pack('=23q', n, b, t, hq, hk, d, d, 8, *[d] * 12, 0, t, 1)
    lib = _native.lib()
    for dtype, code in ((F32, _native.F32), (BF16, _native.BF16)):
        dqw, dkw = (torch.full((n, d), float('nan'), device=DEV, dtype=dtype) for _ in range(2))
        rc = lib.widek_qk_norm_rope_bwd(*[None] * 11, dqw.data_ptr(), dkw.data_ptr(), geom, 1e-6, 0, 0, code, None, 0,
                                        torch.cuda.current_stream().cuda_stream)
        assert rc == _native.WIDEK_OK
        assert float(dqw.abs().max()) == 0.0 and float(dkw.abs().max()) == 0.0
        rc = lib.widek_qk_norm_rope_bwd(*[None] * 13, geom, 1e-6, 0, 0, code, None, 0, None)
        assert rc == _native.WIDEK_OK
