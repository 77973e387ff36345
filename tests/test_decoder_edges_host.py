"""Host-side checks (no GPU) of the decoder-attention operators and their layer
at the edges of what they take."""
import os

import pytest
import torch
from torch.nn.attention import SDPBackend, sdpa_kernel

import decoder_ref as R
import wide_compiler as wc
from conftest import ROOT
from wide_compiler import _autograd as AG


@pytest.mark.parametrize("rows", [4, 0])
@pytest.mark.parametrize("lead", [1, 2, 3])
def test_torch_formulation_treats_positions_past_the_table_as_padding(rows, lead):
    """As the kernel does; on a GPU an index past the table would be a fault."""
    gen = torch.Generator().manual_seed(lead)
    n, b, t, d = 2, 3, 4, 8
    x = torch.randn(n, b, t, 2, d, generator=gen).requires_grad_(True)
    w = (1 + 0.2 * torch.randn(n, d, generator=gen)).requires_grad_(True)
    cos, sin = R.tables(rows, d)
    pos = torch.tensor([0, 4, 2 ** 40, 3]).expand((n, b, t)[3 - lead:])
    valid = torch.where(pos < rows, pos, torch.full_like(pos, -1))
    y, _ = AG.qk_norm_rope_t(x, x.detach(), w, w.detach(), cos, sin, pos, 1e-6, False)
    if rows:
        want, amp = R.rope(x.detach(), w.detach(), cos, sin, valid, 1e-6, False)
        R.assert_within(y.detach(), want, 24 * R.U * amp)
    else:
        assert float(y.detach().abs().max()) == 0.0
    gx, gw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert torch.isfinite(gw).all() and float(gx[:, :, 1:3].abs().max()) == 0.0


def test_torch_formulation_gradient_of_padding_that_holds_nan():
    n, b, t, d = 1, 2, 3, 8
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(n, b, t, 2, d, generator=gen)
    x[:, 0, 1], x[:, 1, 2] = float('nan'), float('inf')
    x.requires_grad_(True)
    w = torch.ones(n, d, requires_grad=True)
    cos, sin = R.tables(4, d)
    pos = torch.tensor([[0, -1, 2], [0, 1, -1]])
    y, _ = AG.qk_norm_rope_t(x, x.detach(), w, w.detach(), cos, sin, pos, 1e-6, False)
    dy = torch.randn(y.shape, generator=gen)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    dx, dw, dx_amp, dw_amp = R.rope_grad(x.detach(), w.detach(), cos, sin, pos, 1e-6, False, dy)
    R.assert_within(gx, dx, 48 * R.U * dx_amp)
    R.assert_within(gw, dw, (24 + b * t * 2) * R.U * dw_amp)


def plain_kernels(monkeypatch):
    """Stands the launches of norm + rotation in with graph-free formulas."""
    from wide_compiler import ops

    def forward(*args):
        with torch.no_grad():
            return AG.qk_norm_rope_t(*args)

    def backward(q, k, qw, kw, cos, sin, pos, dyq, dyk, eps=1e-6, interleaved=False, need_dw=True):
        with torch.enable_grad():
            ins = [x.detach().requires_grad_(True) for x in (q, k, qw, kw)]
            y = AG.qk_norm_rope_t(*ins, cos, sin, pos, eps, interleaved)
            return torch.autograd.grad(y, ins, [dyq.detach(), dyk.detach()])

    monkeypatch.setattr(ops, "_qk_norm_rope", forward)
    monkeypatch.setattr(ops, "qk_norm_rope_bwd", backward)
    return ops


@pytest.mark.parametrize("shared", [False, True])
def test_gradient_penalty_through_norm_and_rotation(monkeypatch, shared):
    """A gradient of a gradient: also where k is computed from q, and where
    only one output is used."""
    ops = plain_kernels(monkeypatch)
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(2, 2, 3, 2, 8, generator=gen).requires_grad_(True)
    w = (1 + 0.2 * torch.randn(2, 8, generator=gen)).requires_grad_(True)
    cos, sin = R.tables(4, 4)
    pos = torch.tensor([0, -1, 3])

    def penalty(f):
        q = x * 1.5
        k = q.tanh() if shared else x[..., :1, :]
        yq, yk = f(q, k, w, w * 0.5, cos, sin, pos, 1e-6, True)
        out = (yq ** 3).sum() + ((yk ** 2).sum() if shared else 0)
        g, = torch.autograd.grad(out, x, create_graph=True)
        return torch.autograd.grad((g ** 2).sum(), (x, w))

    for got, want in zip(penalty(ops.qk_norm_rope), penalty(AG.qk_norm_rope_t)):
        torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-5)


def test_gradient_penalty_through_the_recomputed_attention(monkeypatch):
    """ops.causal_attention's backward is the torch formulation's: with a graph
    where one is asked for."""
    gen = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(1, 2, 5, h, 8, generator=gen).requires_grad_(True) for h in (4, 2, 2))

    def forward(q, k, v):
        with torch.no_grad():
            return AG.causal_attention_t(q, k, v)

    def penalty(f):
        out = f(q, k, v)
        g = torch.autograd.grad((out ** 2).sum(), (q, k, v), create_graph=True)
        return torch.autograd.grad(sum((x ** 2).sum() for x in g), (q, k, v))

    got = penalty(lambda *a: AG.run(forward, AG.causal_attention_t, *a))
    with sdpa_kernel(SDPBackend.MATH):                       # torch's other forms have no second gradient
        plain = penalty(AG.causal_attention_t)
    for got, want in zip(got, plain):
        torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-5)


def test_forward_mode_tangents_are_refused(monkeypatch):
    """The kernels have no forward-mode gradients: a tangent was dropped."""
    import torch.autograd.forward_ad as fwd
    ops = plain_kernels(monkeypatch)
    x, w = torch.randn(1, 1, 2, 1, 8), torch.ones(1, 8)
    cos, sin = R.tables(4, 4)
    pos = torch.arange(2)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for grad in (False, True):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                ops.qk_norm_rope(dual, x, w, w, cos, sin, pos)
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                ops.decode_attention(dual[:, :, 0], None, pos[:1])
        ops.qk_norm_rope(x, x, w, w, cos, sin, pos)


def test_layer_refuses_what_its_positions_do_not_reach():
    """Both lengths are known on the host: past the rotation table keys were
    left out of the cache and then attended over."""
    layer = wc.WideDecoderAttention(1, 32, 4, 2, max_positions=20)
    with pytest.raises(ValueError, match="max_positions"):
        layer.new_cache(2, 21)
    cache = layer.new_cache(2, 20, page_size=16)                 # room for 32 in whole pages
    with pytest.raises(ValueError, match="21 tokens"):
        layer(torch.zeros(1, 2, 21, 32))
    with pytest.raises(ValueError, match="21 tokens"):
        layer.prefill(torch.zeros(1, 2, 21, 32), layer.new_cache(2, 12, page_size=4))
    with pytest.raises(ValueError, match="13 tokens"):
        layer.prefill(torch.zeros(1, 2, 13, 32), layer.new_cache(2, 12, page_size=4))
    with pytest.raises(RuntimeError, match="CUDA"):              # this one fits: only the device is missing
        layer.prefill(torch.zeros(1, 2, 20, 32), cache)


def test_rotation_tables_follow_what_they_are_made_from():
    layer = wc.WideDecoderAttention(1, 32, 4, max_positions=20)
    cpu = torch.device('cpu')
    assert layer.rotation(cpu)[0].shape == (20, 4) and layer.rotation(cpu)[0] is layer.rotation(cpu)[0]
    cos = layer.rotation(cpu, 32)[0]
    assert cos.shape == (32, 4) and torch.equal(cos[:20], layer.rotation(cpu)[0])
    layer.theta = 100.0
    assert not torch.equal(layer.rotation(cpu)[0], cos[:20])
    layer.rotary_dim, layer.max_positions = 4, 7
    assert layer.rotation(cpu)[0].shape == (7, 2)


def test_rotation_tables_first_made_under_inference_mode_can_train():
    layer = wc.WideDecoderAttention(1, 32, 4, max_positions=20)
    with torch.inference_mode():
        cos, sin = layer.rotation(torch.device('cpu'))
    assert not cos.is_inference() and not sin.is_inference()


def test_rotation_tables_are_not_made_during_a_graph_capture(monkeypatch):
    """Their copy to the device cannot be recorded; made before, they serve."""
    layer = wc.WideDecoderAttention(1, 32, 4, max_positions=20)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captur"):
        layer.rotation(torch.device('cuda', 0))


def test_example_takes_prompts_of_no_tokens(monkeypatch):
    """Their row of logits was row -1: on a GPU an index out of range."""
    monkeypatch.syspath_prepend(os.path.join(ROOT, "examples"))
    from wide_decoder import WideDecoder
    model = WideDecoder(2, 10, 16, 1, 2, 1, 8)
    monkeypatch.setattr(model, "prefill", lambda tokens, caches, pos: torch.randn(2, 3, tokens.shape[2], 10))
    monkeypatch.setattr(model, "step", lambda tokens, caches, lengths: torch.randn(2, 3, 1, 10))
    lengths = torch.tensor([[0, 1, 4], [4, 0, 2]], dtype=torch.int32)
    tokens, logits = model.generate(torch.zeros(2, 3, 4, dtype=torch.long), lengths, 5)
    assert tokens.shape == (2, 3, 5) and logits.shape == (2, 3, 5, 10)
    with pytest.raises(ValueError, match="max_len"):
        model.generate(torch.zeros(2, 3, 4, dtype=torch.long), lengths, 6)


def test_workspace_is_asked_for_on_the_tensors_device(monkeypatch):
    """It depends on that GPU's SM count; asked for on the current device, a
    size that another one needs was refused, and remembered."""
    from wide_compiler import _native as N
    from wide_compiler import ops
    at = [0]

    class Device:
        def __init__(self, idx):
            self.idx = idx

        def __enter__(self):
            self.was, at[0] = at[0], self.idx

        def __exit__(self, *_):
            at[0] = self.was

    class Lib:
        @staticmethod
        def query(*args):
            return 100 + at[0]

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(ops, "_current_device", lambda: at[0])
    monkeypatch.setattr(N, "lib", lambda: Lib)
    monkeypatch.setattr(ops, "_WS_BYTES", {})
    for _ in range(2):
        assert ops._workspace("query", 0, ("a", 0), 1) == 100
        assert ops._workspace("query", 3, ("a", 3), 1) == 103
    assert at[0] == 0


def test_gradient_entry_refuses_a_workspace_that_floats_cannot_lie_in():
    import struct

    from wide_compiler import _native as N
    lib = N.load()
    n, b, t, hq, hk, d = 2, 2, 3, 4, 2, 64
    geom = [n, b, t, hq, hk, d, d, 8]
    for h in (hq, hk, hk):
        geom += [b * t * h * d, t * h * d, h * d, d]
    geom = struct.pack('=23q', *geom, 0, t, 1)
    size = lib.widek_qk_norm_rope_bwd_workspace(geom)
    P = 16                               # stand-in pointers: never dereferenced on this path
    rc = lib.widek_qk_norm_rope_bwd(*[P] * 13, geom, 1e-6, 0, 0, N.BF16, P + 2, size, None)
    assert rc == N.WIDEK_ERR_INVALID and "workspace" in N.last_error()


def test_cache_sizes_that_make_no_pages_are_refused():
    for kw in (dict(max_len=8, page_size=0), dict(max_len=8, page_size=-4), dict(max_len=-1, page_size=4)):
        with pytest.raises(ValueError, match="page"):
            wc.WidePagedCache.allocate(1, 2, 1, 8, device='cpu', **kw)
    assert wc.WidePagedCache.allocate(1, 2, 1, 8, max_len=0, page_size=4, device='cpu').max_len == 0
