"""Layers that are turned into 8-bit ones in place, when that fails on the way
(device memory that runs out): a stand-in for the quantiser, no GPU."""
import copy
import pickle

import pytest
import torch

import wide_compiler as wc
from wide_compiler import ops


@pytest.fixture
def quantiser(monkeypatch):
    """ops.quantize_rows in torch, which fails at the calls listed in `fails`."""
    calls = []

    def quantize_rows(x):
        calls.append(x)
        if not x.is_floating_point():
            raise TypeError(f"quantize_rows: {x.dtype}")
        if len(calls) in quantize_rows.fails:
            raise torch.cuda.OutOfMemoryError("no room")
        scale = x.abs().amax(-1).clamp(min=2.0 ** -40) / 127
        return torch.round(x / scale[..., None]).to(torch.int8), scale

    quantize_rows.fails, quantize_rows.calls = (), calls
    monkeypatch.setattr(ops, "quantize_rows", quantize_rows)
    return quantize_rows


@pytest.mark.parametrize("fails", [1, 2])
def test_attention_is_quantised_whole_or_not_at_all(quantiser, fails):
    attn = wc.WideDecoderAttention(2, 32, 4, bias=True)
    before = {k: v.clone() for k, v in attn.state_dict().items()}
    quantiser.fails = (fails,)
    with pytest.raises(torch.cuda.OutOfMemoryError):
        attn.quantize_()
    after = attn.state_dict()
    assert attn.qkv_int8 is None and attn.out_int8 is None
    assert before.keys() == after.keys() and all(torch.equal(before[k], after[k]) for k in before)
    assert attn.qkv_weight.requires_grad
    attn.quantize_()
    assert isinstance(attn.qkv_int8, wc.WideLinearInt8) and isinstance(attn.out_int8, wc.WideLinearInt8)
    assert attn.qkv_weight is None and attn.out_bias is None and not attn.q_norm.requires_grad


@pytest.mark.parametrize("fails", [2, 4, 5, 8])
def test_a_stack_goes_on_where_it_stopped(quantiser, fails):
    """Layers of four products: the layer in which it failed is as it was, and so are the later ones."""
    stack = wc.WideDecoderStack(2, 32, 2, 4, hidden=48, bias=True)
    quantiser.fails = (fails,)
    with pytest.raises(torch.cuda.OutOfMemoryError):
        stack.quantize_()
    done = (fails - 1) // 4
    assert not stack.quantized
    for i, layer in enumerate(stack.layers):
        kinds = {type(layer.up), type(layer.down)}
        assert kinds == {wc.WideLinearInt8 if i < done else wc.WideLinear}
        assert (layer.attn.qkv_int8 is not None) == (layer.attn.out_int8 is not None) == (i < done)
    stack.quantize_()
    assert stack.quantized and not any(p.requires_grad for p in stack.parameters())
    for layer in stack.layers:
        assert {type(m) for m in (layer.up, layer.down, layer.attn.qkv_int8, layer.attn.out_int8)} == {wc.WideLinearInt8}


def test_a_layer_that_was_quantised_before():
    """The layers of a stack may have been quantised one by one."""
    stack = wc.WideDecoderStack(1, 32, 1, 4)
    up = wc.WideLinearInt8(1, 32, 128, bias=False)
    stack.layers[0].up, stack.layers[0].down = up, wc.WideLinearInt8(1, 128, 32, bias=False)
    stack.layers[0].attn.qkv_int8, stack.layers[0].attn.out_int8 = wc.WideLinearInt8(1, 32, 96), wc.WideLinearInt8(1, 32, 32)
    assert stack.quantize_().layers[0].up is up and stack.quantized


def test_layers_pickled_before_there_were_8_bit_projections():
    """They lack the attributes that came with quantize_()."""
    attn = wc.WideDecoderAttention(2, 32, 4)
    state = {k: v for k, v in attn.__dict__.items() if k not in ('qkv_int8', 'out_int8')}
    old = wc.WideDecoderAttention.__new__(wc.WideDecoderAttention)
    old.__setstate__(state)
    assert old.qkv_int8 is None and old.out_int8 is None
    with pytest.raises(TypeError, match="quantise"):
        old((torch.zeros(2, 1, 3, 32, dtype=torch.int8), torch.ones(2, 1, 3)))
    assert wc.WideDecoderAttention.from_modules([old, attn]).n == 4


def test_quantised_layers_are_copied_and_pickled(quantiser):
    attn = wc.WideDecoderAttention(2, 32, 4).quantize_()
    for other in (copy.deepcopy(attn), pickle.loads(pickle.dumps(attn))):
        assert torch.equal(other.qkv_int8.weight, attn.qkv_int8.weight) and other.qkv_weight is None
        assert other.qkv_int8 is not attn.qkv_int8 and other.quantize_() is other
