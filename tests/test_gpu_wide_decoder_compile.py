"""The decoder-attention operators under torch.compile."""
import pytest
import torch

import decoder_ref as R
import wide_compiler as wc
from gpu_util import FP32_TOL
from wide_compiler import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.grad
def test_operators_under_torch_compile():
    torch.manual_seed(5)
    n, b, t, hq, hk, d = 2, 2, 3, 4, 2, 64
    q, k, v = (torch.randn(n, b, t, h, d, device=DEV) for h in (hq, hk, hk))
    w = 1 + 0.2 * torch.randn(n, d, device=DEV)
    cos, sin = (x.to(DEV) for x in R.tables(8, d))
    pos = torch.arange(t, device=DEV)
    f = torch.compile(lambda q, k, w: ops.qk_norm_rope(q, k, w, w, cos, sin, pos), fullgraph=True, backend="eager")
    for x, y in zip(f(q, k, w), ops.qk_norm_rope(q, k, w, w, cos, sin, pos)):
        assert torch.equal(x, y)
    qg, wg = q.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dy = torch.randn_like(q)
    got = torch.autograd.grad(f(qg, k, wg)[0], (qg, wg), dy)
    want = torch.autograd.grad(ops.qk_norm_rope(qg, k, wg, wg, cos, sin, pos)[0], (qg, wg), dy)
    for x, y in zip(got, want):
        torch.testing.assert_close(x, y, **FP32_TOL)

    def held():
        return wc.WidePagedCache.allocate(n, b, hk, d, 8, 4, torch.float32, DEV)

    def step(cache, q, k, v, lengths):
        q = ops.qk_norm_rope_write(q, k, v, w, w, cos, sin, pos, cache)
        return ops.decode_attention(q[:, :, -1], cache, lengths)

    lengths = torch.tensor([3, 2], device=DEV, dtype=torch.int32)
    c1, c2 = held(), held()
    with torch.no_grad():
        want = step(c1, q, k, v, lengths)
        got = torch.compile(step, backend="eager")(c2, q, k, v, lengths)
        assert torch.equal(got, want)
        kr, vr = torch.compile(lambda c: ops.cache_read(c, pos), backend="eager")(c2)
        assert torch.equal(kr, ops.cache_read(c1, pos)[0]) and torch.equal(vr, ops.cache_read(c1, pos)[1])
