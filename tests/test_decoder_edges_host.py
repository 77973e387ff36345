"""Host-side checks (no GPU) of the decoder-attention operators and their layer
at the edges of what they take."""
import pytest
import torch

import decoder_ref as R
import wide_compiler as wc
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
