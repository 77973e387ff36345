"""Refusals of the block-boundary operators: arguments are checked before any
device call, so no GPU is needed."""
import math
import pathlib
import re

import numpy as np
import pytest
import torch

from wide_compiler import _native as N
from wide_compiler import ops

P = 1024                                 # a stand-in pointer: never dereferenced on these paths


def rnorm(x=P, y=P, w=P, wb=None, pw=None, pb=None, gate=None, h=P, z=P, stats=None, n=2, rows=6, d=64, gate_rows=-1,
          scale=1.0, eps=1e-6, center=0, dtype=N.BF16):
    return N.lib().widek_residual_norm_fwd(x, y, w, wb, pw, pb, gate, h, z, stats, n, rows, d, gate_rows, scale, eps,
                                           center, dtype, None)


@pytest.mark.parametrize("bad, word", [
    (dict(n=-1), "sizes"), (dict(rows=-1), "sizes"), (dict(d=0), "sizes"), (dict(d=8193), "8192"),
    (dict(dtype=9), "dtype"), (dict(n=3, rows=0x40000000), "2^31"), (dict(gate=P, gate_rows=4), "gate"),
    (dict(gate=P), "gate"), (dict(gate_rows=6), "gate"), (dict(y=None, pw=P), "no y"),
    (dict(y=None, gate=P, gate_rows=6), "no y"), (dict(pb=P, center=1), "without its weight"), (dict(wb=P), "LayerNorm"),
    (dict(pw=P, pb=P), "LayerNorm"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(z=None), "null"),
    (dict(h=None), "null"), (dict(stats=P + 4), "border")])
def test_forward_refuses(bad, word):
    assert rnorm(**bad) == N.WIDEK_ERR_INVALID
    assert word in N.last_error()


def test_no_rows_is_no_call():
    assert rnorm(x=None, y=None, w=None, h=None, z=None, n=0) == 0
    assert rnorm(x=None, y=None, w=None, h=None, z=None, rows=0) == 0
    assert N.lib().widek_quantize_rows_fwd(None, None, None, 0, 7, 16, N.F32, None) == 0


def test_codes_refuse():
    lib = N.lib()
    call = lambda ld, codes=P, d=64: lib.widek_residual_norm_quantize_fwd(
        P, P, P, None, None, None, None, P, codes, P, ld, 2, 6, d, -1, 1.0, 1e-6, 0, N.BF16, None)
    for args in ((60,), (72,), (64, P + 8)):
        assert call(*args) == N.WIDEK_ERR_INVALID
        assert "16 bytes" in N.last_error()
    quant = lambda rows=3, d=64, ld=64, x=P, scales=P, dtype=N.F32: lib.widek_quantize_rows_fwd(
        x, P, scales, rows, d, ld, dtype, None)
    for bad in (dict(rows=-1), dict(d=-1), dict(ld=63), dict(ld=72), dict(x=None), dict(scales=None), dict(dtype=7)):
        assert quant(**bad) == N.WIDEK_ERR_INVALID


def test_backward_refuses(monkeypatch):
    lib = N.lib()
    assert lib.widek_residual_norm_bwd_workspace(2, 6, 0, -1, 0, 0) == -1
    assert lib.widek_residual_norm_bwd_workspace(2, 6, 9000, -1, 0, 0) == -1

    def bwd(y=P, pw=None, gate=None, stats=P, dy=None, dwb=None, dpw=None, dpb=None, dgate=None, n=2, rows=6, d=64,
            gate_rows=-1, center=0, ws=P, ws_bytes=1 << 30):
        return lib.widek_residual_norm_bwd(P, y, P, None, pw, None, gate, stats, P, P, P, dy, P, dwb, dpw, dpb, dgate, n,
                                           rows, d, gate_rows, 1.0, 1e-6, center, N.BF16, ws, ws_bytes, None)

    for bad, word in ((dict(y=None, dy=P), "not there"), (dict(dpw=P), "not there"), (dict(dgate=P), "not there"),
                      (dict(dwb=P), "not there"), (dict(ws=None), "workspace"), (dict(ws_bytes=8), "workspace"),
                      (dict(ws=P + 2), "workspace"), (dict(stats=None), "statistics"), (dict(stats=P + 8), "statistics")):
        assert bwd(**bad) == N.WIDEK_ERR_INVALID
        assert word in N.last_error(), bad
    assert bwd(rows=0) == 0


def test_operators_refuse_cpu_tensors():
    x, w = torch.zeros(2, 3, 8), torch.ones(2, 8)
    for call in (lambda: ops.residual_norm(x, x, w), lambda: ops.residual_norm_quantize(x, x, w),
                 lambda: ops.quantize_rows(x)):
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_operators_refuse_gradients_they_do_not_have():
    x, w = torch.zeros(2, 3, 8, requires_grad=True), torch.ones(2, 8)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.residual_norm_quantize(x, x, w)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.quantize_rows(x)


@pytest.mark.parametrize("change, error, word", [
    (dict(y=(2, 3, 9)), ValueError, "does not match"), (dict(weight=(8,)), ValueError, "weight"),
    (dict(weight=(3, 8)), ValueError, "weight"), (dict(post_weight=(2, 7)), ValueError, "post_weight"),
    (dict(gate=(8,)), ValueError, "gate"), (dict(gate=(2, 2, 8)), ValueError, "gate"),
    (dict(gate=(2, 3, 1, 8)), ValueError, "gate"), (dict(gate=(2, 3, 1)), ValueError, "gate"),
    (dict(x=(8,), y=(8,)), ValueError, "x must be")])
def test_shapes_are_checked(change, error, word, monkeypatch):
    monkeypatch.setattr(ops, "_device", lambda what, ref, *others: 0)
    shapes = dict(dict(x=(2, 3, 8), y=(2, 3, 8), weight=(2, 8)), **change)
    with torch.no_grad(), pytest.raises(error, match=word):
        ops.residual_norm(**{k: torch.zeros(s) for k, s in shapes.items()})


def test_types_are_checked(monkeypatch):
    monkeypatch.setattr(ops, "_device", lambda what, ref, *others: 0)
    x, w = torch.zeros(2, 3, 8), torch.ones(2, 8)
    with torch.no_grad(), pytest.raises(TypeError, match="mismatch"):
        ops.residual_norm(x, x, w.half())
    with torch.no_grad(), pytest.raises(TypeError, match="support"):
        ops.quantize_rows(torch.zeros(2, 8, dtype=torch.int32))


# ---------------------------------------------------------------------------
# 8-bit linear layers
# ---------------------------------------------------------------------------

def int8(a=P, sa=P, w=P, sw=P, y=P, n=2, m=3, k=64, o=5, a_ld=64, a_ms=192, w_ld=64, w_ms=320, act=0, dtype=N.BF16):
    return N.lib().widek_linear_int8_fwd(a, sa, w, sw, None, y, n, m, k, o, a_ld, a_ms, w_ld, w_ms, act, dtype, None)


@pytest.mark.parametrize("bad, word", [
    (dict(n=-1), "sizes"), (dict(m=-1), "sizes"), (dict(k=0), "sizes"), (dict(k=131072, a_ld=131072, w_ld=131072), "131071"),
    (dict(o=-1), "sizes"), (dict(act=3), "activation"), (dict(dtype=5), "dtype"), (dict(a=None), "null"),
    (dict(sa=None), "null"), (dict(w=None), "null"), (dict(sw=None), "null"), (dict(y=None), "null"),
    (dict(a=P + 8), "16 bytes"), (dict(w=P + 1), "16 bytes"), (dict(a_ld=72), "16 bytes"), (dict(w_ld=48), "16 bytes"),
    (dict(a_ms=8), "16 bytes"), (dict(w_ms=-16), "16 bytes"), (dict(m=1 << 40), "tiles"), (dict(o=1 << 33), "tiles")])
def test_linear_int8_refuses(bad, word):
    assert int8(**bad) == N.WIDEK_ERR_INVALID
    assert word in N.last_error()


def test_linear_int8_of_nothing():
    for size in ("n", "m", "o"):
        assert int8(**{size: 0}) == 0


@pytest.mark.parametrize("change, error", [
    (dict(codes=(2, 3, 17)), ValueError), (dict(codes=(3, 3, 16)), ValueError), (dict(codes=(16,)), ValueError),
    (dict(weight=(2, 16)), ValueError), (dict(scale=(2, 4)), ValueError), (dict(weight_scale=(2, 4)), ValueError),
    (dict(bias=(2, 6)), ValueError)])
def test_linear_int8_checks_shapes(change, error, monkeypatch):
    monkeypatch.setattr(ops, "_device", lambda what, ref, *others: 0)
    shapes = dict(dict(codes=(2, 3, 16), scale=(2, 3), weight=(2, 5, 16), weight_scale=(2, 5), bias=(2, 5)), **change)
    args = {k: torch.zeros(s, dtype=torch.int8 if k in ("codes", "weight") else torch.float32) for k, s in shapes.items()}
    with torch.no_grad(), pytest.raises(error, match="linear_int8"):
        ops.linear_int8(**args, dtype=torch.float32)


def test_linear_int8_checks_types(monkeypatch):
    monkeypatch.setattr(ops, "_device", lambda what, ref, *others: 0)
    i8 = lambda *s: torch.zeros(s, dtype=torch.int8)
    f = lambda *s: torch.zeros(s)
    with pytest.raises(TypeError, match="int8"):
        ops.linear_int8(f(2, 3, 16), f(2, 3), i8(2, 5, 16), f(2, 5))
    with pytest.raises(TypeError, match="float32"):
        ops.linear_int8(i8(2, 3, 16), f(2, 3).half(), i8(2, 5, 16), f(2, 5))
    with pytest.raises(ValueError, match="bias"):
        ops.linear_int8(i8(2, 3, 16), f(2, 3), i8(2, 5, 16), f(2, 5), f(2, 5), dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="support"):
        ops.linear_int8(i8(2, 3, 16), f(2, 3), i8(2, 5, 16), f(2, 5), dtype=torch.float64)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.linear_int8(i8(2, 3, 16), f(2, 3).requires_grad_(), i8(2, 5, 16), f(2, 5))


def test_rows_of_codes_read_in_place_or_copied():
    i8 = lambda *s: torch.zeros(s, dtype=torch.int8)
    base = i8(4096)                                   # 64-byte aligned
    at = lambda t, *shape: base[t:t + torch.Size(shape).numel()].view(shape)
    for t, ld, ms in ((at(0, 2, 3, 32), 32, 96), (at(0, 2, 3, 4, 48)[..., :40], 48, 576), (at(0, 1, 1, 7), 16, 16),
                      (at(0, 2, 6, 32)[:, ::2], 64, 192), (at(16, 4, 64)[..., :50], 64, 64)):
        got = ops._rows16(t)
        assert got[0] is t and got[1:] == (ld, ms)
    for t in (at(0, 2, 3, 33), at(0, 2, 3, 4, 32).transpose(1, 2), at(0, 2, 33, 3).transpose(1, 2), at(1, 2, 3, 32),
              at(0, 1, 5, 16).expand(3, -1, -1), at(0, 2, 1, 32).expand(-1, 5, -1)):
        got, ld, ms = ops._rows16(t)
        assert got is not t and got.shape == t.shape and ld % 16 == 0 and ms == ld * t[0].numel() // t.shape[-1]


def test_gelu_of_16_bit_results():
    """fp32 restatement of Gelu2 in csrc/linear_int8.cu with the coefficients read
    from it: the normal tail within 9e-6 of itself up to 8."""
    src = (pathlib.Path(ops.__file__).resolve().parents[1] / "csrc" / "linear_int8.cu").read_text()
    body = src[src.index("constexpr float c[9] = {"):]
    r = np.float32([float(v) for v in re.findall(r"(-?[0-9.]+(?:e-[0-9]+)?)f", body[body.index("{"):body.index("}")])])
    assert len(r) == 9
    a = np.linspace(0, 8, 200001).astype(np.float32)
    f32 = lambda v: v.astype(np.float32)
    p = np.full_like(a, r[8])
    for c in r[7::-1]:
        p = f32(p.astype(np.float64) * a + c)                    # fused: one rounding
    e = f32(f32(a * np.float32(-0.72134752)).astype(np.float64) * a + p)
    tail = np.array([math.erfc(float(v) / math.sqrt(2)) / 2 for v in a])
    # the exponent's own roundings: 2 of at most 46 * 2^-24
    assert np.abs(np.exp2(e.astype(np.float64)) / tail - 1).max() < 9e-6 + 2 * 46 * 2.0 ** -24 * math.log(2)


# ---------------------------------------------------------------------------
# Modules and torch.library operators
# ---------------------------------------------------------------------------

def test_fake_implementations():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from wide_compiler import _autograd as AG
    w = torch.ops.widek
    with FakeTensorMode():
        t = lambda *s, dt=torch.bfloat16: torch.empty(*s, device='cuda', dtype=dt)
        x, nd, gate = t(2, 3, 5, 40), t(2, 40), t(2, 3, 40)
        same = lambda a, b: all(p.shape == q.shape and p.dtype == q.dtype and p.device == q.device for p, q in zip(a, b))
        assert same(w.residual_norm(x, x, nd, None, nd, None, gate, 1.0, 1e-6, False),
                    AG.residual_norm_t(x, x, nd, None, nd, None, gate, 1.0, 1e-6, False))
        assert w.row_norm(x, nd, nd, 1e-6, True).shape == x.shape
        for codes, scale in (w.quantize_rows(x), w.row_norm_quantize(x, nd, None, 1e-6, False),
                             w.residual_norm_quantize(x, x, nd, None, None, None, None, 1.0, 1e-6, False)[1:]):
            assert codes.shape == x.shape and codes.dtype == torch.int8 and codes.stride(-2) == 48
            assert scale.shape == x.shape[:-1] and scale.dtype == torch.float32
        y = w.linear_int8(codes, scale, t(2, 7, 40, dt=torch.int8), t(2, 7, dt=torch.float32), None, 0, torch.float16)
        assert y.shape == (2, 3, 5, 7) and y.dtype == torch.float16


def test_stack_is_built_and_refuses():
    import wide_compiler as wc
    s = wc.WideDecoderStack(2, 32, 3, 4, 2, norm='layer', post_norm=True, gate_init=0.1, max_positions=9)
    names = {k for k, _ in s.named_parameters()}
    assert {'layers.2.attn_gate', 'layers.0.mlp_post.bias', 'norm.bias', 'layers.1.up.weight'} <= names
    assert s.layers[0].attn.max_positions == 9 and 'layers=3' in repr(s)
    plain = wc.WideDecoderStack(2, 32, 1, 4)
    assert not any('bias' in k or 'gate' in k or 'post' in k for k in plain.state_dict())
    with pytest.raises(ValueError, match="norm must be"):
        wc.WideDecoderStack(2, 32, 1, 4, norm='batch')
    with pytest.raises(ValueError, match="input must be"):
        s(torch.zeros(2, 3, 32))
    with pytest.raises(ValueError, match="gates for 3 layers"):
        s(torch.zeros(2, 1, 3, 32), gates=[torch.zeros(2, 32)])


def test_codes_need_a_quantised_layer():
    import wide_compiler as wc
    attn = wc.WideDecoderAttention(2, 32, 4)
    with pytest.raises(TypeError, match="quantise"):
        attn((torch.zeros(2, 1, 3, 32, dtype=torch.int8), torch.ones(2, 1, 3)))


def test_int8_layer_keeps_its_scales_when_cast():
    import wide_compiler as wc
    layer = wc.WideLinearInt8(2, 17, 5)
    layer.weight_scale.fill_(1 / 3)
    for bias in (True, False):
        layer = wc.WideLinearInt8(2, 17, 5, bias)
        layer.weight_scale.fill_(1 / 3)
        want = layer.weight_scale.clone()
        layer.to(torch.float16)
        assert layer.dtype == torch.float16 and torch.equal(layer.weight_scale, want)
        assert layer.codes.shape == (2, 5, 17) and layer.codes.stride(1) == 32
        layer.to(torch.float32)
        assert layer.dtype == torch.float32 and layer.weight_scale.dtype == torch.float32
