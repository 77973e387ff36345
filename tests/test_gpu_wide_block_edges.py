"""The block-boundary operators at the edges of their sizes, and the 8-bit linear
layer's kernels beside one another."""
import pytest
import torch

from gpu_util import no_device_error
from wide_compiler import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def int8_case(n, m, k, o, seed=0):
    gen = torch.Generator().manual_seed(seed)
    ints = lambda *s: torch.randint(-127, 128, s, generator=gen, dtype=torch.int8).to(DEV)
    return ints(n, m, k), torch.rand(n, m, generator=gen).to(DEV), ints(n, o, k), torch.rand(n, o, generator=gen).to(DEV)


def test_parts_of_k_beside_wide_tiles():
    """Few tokens with K over a cluster (8, 4 and 2 parts) on one stream, 256 x 256 tiles of block pairs on
    another: the results of each alone."""
    few = [int8_case(1, 1, 8192, 512), int8_case(1, 33, 4096, 1024), int8_case(2, 100, 2048, 512)]
    many = [int8_case(4, 1024, 512, 1024), int8_case(1, 4096, 1024, 2048)]
    want = [[ops.linear_int8(*a, dtype=BF16) for a in side] for side in (few, many)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for i in range(30):
        for side, (cases, stream) in enumerate(zip((few, many), streams)):
            with torch.cuda.stream(stream):
                outs[side] += [ops.linear_int8(*a, dtype=BF16) for a in cases]
    torch.cuda.synchronize()
    for side, out in enumerate(outs):
        assert all(torch.equal(y, want[side][i % len(want[side])]) for i, y in enumerate(out))
    no_device_error()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows", [1, 3, 4000])
@pytest.mark.parametrize("post", [False, True])
def test_codes_of_one_channel_under_a_layer_norm(rows, post, dtype):
    """A single channel is its own mean: v - mean is exactly 0, and 0 * factor * weight + bias is exactly the
    bias. So z == bias, scale = max(|bias|, 2^-40) / 127 in fp32, code = +-127 or, for no bias, 0."""
    gen = torch.Generator().manual_seed(rows)
    n = 5
    x, y = ((3 * torch.randn(n, rows, 1, generator=gen)).to(dtype).to(DEV) for _ in range(2))
    weight = (1 + 0.3 * torch.randn(n, 1, generator=gen)).to(dtype).to(DEV)
    bias = torch.tensor([[0.3], [-1.7], [0.0], [5.0], [-2.0 ** -14]]).to(dtype).to(DEV)
    pw, pb = (weight, bias.flip(0).contiguous()) if post else (None, None)
    want = bias.float()[:, None].expand(n, rows, 1)
    top = want.abs().amax(-1).clamp(min=2.0 ** -40)
    scale = top / torch.full_like(top, 127.0)
    h, z = ops.residual_norm(x, y, weight, bias, pw, pb, center=True)
    h8, codes, scales = ops.residual_norm_quantize(x, y, weight, bias, pw, pb, center=True)
    assert torch.equal(z.float(), want) and torch.equal(h, h8)
    assert torch.equal(scales, scale)
    assert torch.equal(codes.float(), torch.round(want / scale.unsqueeze(-1)))
    assert codes.float().abs().amax() == 127 and not codes[2].any()
    u = pb.float()[:, None] if post else y.float()
    assert torch.equal(h, (x.float() + u).to(dtype))
    no_device_error()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n, m, k, o", [(1, 129, 16, 16), (1, 129, 64, 8), (1, 130, 333, 517), (2, 257, 1040, 130), (1, 300, 1920, 96),
                                        (1, 256, 2048, 256), (1, 511, 4096, 300), (3, 140, 2000, 1000), (2, 129, 16384, 1500)])
def test_more_rows_than_narrow_tiles_and_few_tiles(n, m, k, o, dtype):
    """Single 256 x 256 tiles and K in parts on both sides of the rule between them: the exact sum with its
    scales, and the same rows 100 at a time (narrow tiles of one block of rows) to the bit."""
    codes, scale, w, ws = int8_case(n, m, k, o, m + k)
    y = ops.linear_int8(codes, scale, w, ws, act=ops.ACT_RELU, dtype=dtype)
    acc = torch.matmul(codes.double().cpu(), w.double().cpu().transpose(1, 2))
    want = (acc * scale.double().cpu().unsqueeze(-1) * ws.double().cpu()[:, None]).clamp(min=0)
    # rounded to fp32, times two scales (each half a step of 2^-24), and to the type (subnormals: half a step of those)
    bound = want * (3 * 2.0 ** -24 * (1 + 2.0 ** -20) + torch.finfo(dtype).eps / 2) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    y64 = y.double().cpu()
    most = torch.finfo(dtype).max
    assert ((y64 - want).abs() <= bound)[want < most].all() and (y64[want > most * 1.001] == float("inf")).all()
    parts = [ops.linear_int8(codes[:, i:i + 100], scale[:, i:i + 100], w, ws, act=ops.ACT_RELU, dtype=dtype) for i in range(0, m, 100)]
    assert torch.equal(torch.cat(parts, 1), y)
    no_device_error()


@pytest.mark.parametrize("n, m, k, o", [(1, 540000, 48, 4096), (1, 540000, 48, 4097), (300000, 8, 16, 1024)])
def test_products_past_32_bits(n, m, k, o):
    """Over 2^31 results (wide tiles by whole vectors and value by value, narrow ones of many models): the last
    rows are what a call on them alone gives."""
    gen = torch.Generator(device=DEV).manual_seed(n + o)
    ints = lambda *s: torch.randint(-127, 128, s, generator=gen, dtype=torch.int8, device=DEV)
    codes, w = ints(n, m, k), ints(n, o, k)
    scale, ws = torch.rand(n, m, generator=gen, device=DEV), torch.rand(n, o, generator=gen, device=DEV)
    y = ops.linear_int8(codes, scale, w, ws, dtype=BF16)
    alone = ops.linear_int8(codes[-1:, -5:], scale[-1:, -5:], w[-1:], ws[-1:], dtype=BF16)
    assert torch.equal(y[-1:, -5:], alone)
    no_device_error()


@pytest.mark.grad
def test_gradients_past_32_bits():
    """Rows of over 2^31 values: the last rows' gradients are those of a call on them alone."""
    n, rows, d = 1, 270000, 8192
    x, y, dh, dz = (torch.randn(n, rows, d, device=DEV, dtype=BF16) for _ in range(4))
    w = 1 + 0.2 * torch.randn(n, d, device=DEV, dtype=BF16)
    need = (True, True) + (False,) * 5

    def grads(x, y, dh, dz):
        _, _, stats, _ = ops._residual_norm(x, y, w, None, w, None, None, 1.0, 1e-6, False, True)
        return ops.residual_norm_bwd(x, y, w, None, w, None, None, stats, dh, dz, need=need)[:2]

    got = grads(x, y, dh, dz)
    want = grads(*(t[:, -5:].contiguous() for t in (x, y, dh, dz)))
    for a, b in zip(got, want):
        # the forward's statistics are summed in another order for few rows: the factors are off by 90 * 2^-24 of
        # themselves, terms of up to 6 by 4e-5; each side is rounded to bf16 once, by up to 2^-8 of its value
        torch.testing.assert_close(a[:, -5:].float(), b.float(), rtol=2.0 ** -7, atol=1e-4)
    no_device_error()
