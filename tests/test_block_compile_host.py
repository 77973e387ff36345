"""What the block-boundary operators refuse, they refuse under torch.compile too."""
import pytest
import torch

from wide_compiler import ops


@pytest.mark.parametrize("part", ["post_weight", "post_bias", "gate"])
@pytest.mark.parametrize("op", [ops.residual_norm, ops.residual_norm_quantize])
def test_parts_of_y_without_y(op, part, monkeypatch):
    """A norm or gate of a block's output that is not there is refused, not left out."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with torch.no_grad(), pytest.raises(ValueError, match="no y"):
        torch.compile(lambda x, w, p: op(x, None, w, center=True, **{part: p}), backend="eager")(
            torch.ones(2, 3, 8), torch.ones(2, 8), torch.ones(2, 8))
    torch._dynamo.reset()
    monkeypatch.setattr(ops, "_compiling", lambda: True)
    with FakeTensorMode(), torch.no_grad():
        x, w = torch.empty(2, 3, 8, device='cuda'), torch.empty(2, 8, device='cuda')
        assert op(x, None, w)[0] is x
        with pytest.raises(ValueError, match="no y"):
            op(x, None, w, center=True, **{part: w})
