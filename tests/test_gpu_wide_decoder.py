"""GPU parity of the decoder-attention operators (norm + rotation with its
gradients, the paged cache, attention of one new token) against the 64-bit
formulas of decoder_ref, with the bounds derived there."""
import math

import pytest
import torch

import decoder_ref as R
import wide_compiler as wc
from gpu_util import no_device_error
from wide_compiler import _native, ops

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
I8, E4M3 = torch.int8, torch.float8_e4m3fn
ROW_OPS = 24          # fp32 roundings on the way to one normed, rotated channel


def heads(n, b, t, hq, hk, d, dtype, gen, fused=True):
    """q, k, v as views of one projection (or dense)."""
    x = (torch.randn(n, b, t, hq + 2 * hk, d, generator=gen) * 1.5).to(dtype).to(DEV)
    if not fused:
        return x[..., :hq, :].contiguous(), x[..., hq:hq + hk, :].contiguous(), x[..., hq + hk:, :].contiguous()
    flat = x.view(n, b, t, -1)
    cut = lambda a, h: flat[..., a * d:(a + h) * d].unflatten(-1, (h, d))
    return cut(0, hq), cut(hq, hk), cut(hq + hk, hk)


def weights(n, d, dtype, gen):
    return (1 + 0.3 * torch.randn(n, d, generator=gen)).to(dtype).to(DEV)


# n, b, t, hq, hk, d, rot: sizes where the vector width, the lanes of a row
# and the share of rotated channels change
ROPE = [
    (2, 3, 5, 4, 2, 64, 64), (1, 1, 1, 1, 1, 128, 128), (3, 2, 7, 6, 3, 128, 32), (2, 1, 9, 8, 1, 80, 40),
    (1, 2, 33, 3, 3, 256, 256), (2, 2, 3, 2, 1, 96, 48), (1, 3, 4, 5, 5, 46, 10), (2, 1, 6, 2, 2, 33, 32),
    (1, 1, 130, 16, 4, 16, 16), (1, 2, 2, 1, 1, 2, 2), (2, 2, 2, 2, 2, 72, 18), (1, 1, 3, 2, 1, 1, 0),
    (2, 2, 4, 3, 1, 250, 124),
]


@pytest.mark.parametrize("shape", ROPE)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_qk_norm_rope(shape, dtype, interleaved):
    n, b, t, hq, hk, d, rot = shape
    gen = torch.Generator().manual_seed(sum(shape))
    q, k, _ = heads(n, b, t, hq, hk, d, dtype, gen)
    qw, kw = weights(n, d, dtype, gen), weights(n, d, dtype, gen)
    cos, sin = R.tables(t + 5, rot)
    pos = torch.randint(-1, t + 5, (n, b, t), generator=gen, dtype=torch.int32)
    yq, yk = ops.qk_norm_rope(q, k, qw, kw, cos.to(DEV), sin.to(DEV), pos.to(DEV), 1e-6, interleaved)
    for y, x, w in ((yq, q, qw), (yk, k, kw)):
        assert y.is_contiguous() and y.dtype == dtype
        want, amp = R.rope(x, w, cos, sin, pos, 1e-6, interleaved)
        R.assert_within(y, want, ROW_OPS * R.U * amp + R.store_ulp(dtype) * want.abs() + R.tiny(dtype))
    no_device_error()


@pytest.mark.parametrize("lead", [1, 2, 3])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_positions_shared_by_leading_dims(lead, itype):
    n, b, t, d = 2, 3, 4, 64
    gen = torch.Generator().manual_seed(lead)
    q, k, _ = heads(n, b, t, 2, 1, d, BF16, gen, fused=False)
    qw = weights(n, d, BF16, gen)
    cos, sin = R.tables(9, d)
    pos = torch.randint(0, 9, (n, b, t)[3 - lead:], generator=gen, dtype=itype)
    yq, _ = ops.qk_norm_rope(q, k, qw, qw, cos.to(DEV), sin.to(DEV), pos.to(DEV))
    want, amp = R.rope(q, qw, cos, sin, pos, 1e-6, False)
    R.assert_within(yq, want, ROW_OPS * R.U * amp + R.store_ulp(BF16) * want.abs())


def test_other_strides_and_offsets():
    """Heads before tokens, a transposed batch and a base that no 16-byte
    vector starts at give what dense copies give."""
    gen = torch.Generator().manual_seed(7)
    n, b, t, h, d = 2, 3, 5, 4, 64
    cos, sin = (x.to(DEV) for x in R.tables(t, d))
    w = weights(n, d, BF16, gen)
    pos = torch.arange(t, device=DEV)
    base = torch.randn(n * b * t * h * d + 3, generator=gen).to(BF16).to(DEV)
    for x in (base[3:].view(n, b, t, h, d), base[:-3].view(n, b, h, t, d).transpose(2, 3),
              base[:-3].view(b, n, t, h, d).transpose(0, 1), base[:-3].view(n, b, t, h, d).flip(2)[:, :, ::2].flip(2)):
        dense = x.contiguous()
        p = pos[:x.shape[2]]
        got, ref = ops.qk_norm_rope(x, x, w, w, cos, sin, p), ops.qk_norm_rope(dense, dense, w, w, cos, sin, p)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_zero_rows_and_padding_that_holds_nan():
    n, b, t, d = 1, 2, 3, 128
    gen = torch.Generator().manual_seed(3)
    q, k, _ = heads(n, b, t, 2, 1, d, F32, gen, fused=False)
    q[:, 0, 1] = 0.0                                  # a row of zeros: r = 1/sqrt(eps), output 0
    q[:, 1, 2] = float('nan')
    k[:, 1, 2] = float('inf')
    w = weights(n, d, F32, gen)
    cos, sin = (x.to(DEV) for x in R.tables(t, d))
    pos = torch.tensor([[0, 1, 2], [0, 1, -1]], device=DEV)
    yq, yk = ops.qk_norm_rope(q, k, w, w, cos, sin, pos)
    assert torch.isfinite(yq).all() and torch.isfinite(yk).all()
    assert float(yq[:, 1, 2].abs().max()) == 0.0 and float(yk[:, 1, 2].abs().max()) == 0.0
    assert float(yq[:, 0, 1].abs().max()) == 0.0
    dq, dk, dqw, dkw = ops.qk_norm_rope_bwd(q, k, w, w, cos, sin, pos, torch.ones_like(yq),
                                            torch.full_like(yk, 1.0).index_fill(2, torch.tensor([2], device=DEV), 1.0))
    for g in (dq, dk, dqw, dkw):
        assert torch.isfinite(g).all()
    assert float(dq[:, 1, 2].abs().max()) == 0.0 and float(dk[:, 1, 2].abs().max()) == 0.0


def test_position_past_the_table_is_an_index_error():
    gen = torch.Generator().manual_seed(4)
    q, k, _ = heads(1, 1, 3, 1, 1, 64, F32, gen)
    w = weights(1, 64, F32, gen)
    cos, sin = (x.to(DEV) for x in R.tables(4, 64))
    yq, _ = ops.qk_norm_rope(q, k, w, w, cos, sin, torch.tensor([0, 4, 3], device=DEV))
    assert _native.device_error() == _native.DEV_ERR_INDEX
    assert float(yq[:, :, 1].abs().max()) == 0.0 and float(yq[:, :, 2].abs().max()) > 0.0


@pytest.mark.grad
@pytest.mark.parametrize("shape", ROPE)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_qk_norm_rope_gradients(shape, dtype, interleaved):
    n, b, t, hq, hk, d, rot = shape
    gen = torch.Generator().manual_seed(sum(shape) + 1)
    q, k, _ = heads(n, b, t, hq, hk, d, dtype, gen)
    ins = [x.detach().requires_grad_(True) for x in (q, k, weights(n, d, dtype, gen), weights(n, d, dtype, gen))]
    cos, sin = R.tables(t + 5, rot)
    pos = torch.randint(-1, t + 5, (b, t), generator=gen)
    dy = [torch.randn(x.shape, generator=gen).to(dtype).to(DEV) for x in (q, k)]
    y = ops.qk_norm_rope(*ins, cos.to(DEV), sin.to(DEV), pos.to(DEV), 1e-6, interleaved)
    got = torch.autograd.grad(y, ins, dy)
    for i in range(2):
        dx, dw, dx_amp, dw_amp = R.rope_grad(ins[i], ins[2 + i], cos, sin, pos, 1e-6, interleaved, dy[i])
        rows = b * t * (hq, hk)[i]
        R.assert_within(got[i], dx, 2 * ROW_OPS * R.U * dx_amp + R.store_ulp(dtype) * dx.abs() + R.tiny(dtype), "dx")
        # one row's term, then a sum over the rows that no order rounds by more than rows * U
        R.assert_within(got[2 + i], dw, (ROW_OPS + rows) * R.U * dw_amp + R.store_ulp(dtype) * dw.abs()
                        + R.tiny(dtype), "dw")


@pytest.mark.grad
def test_qk_norm_rope_gradient_against_differences():
    """The 64-bit gradient formulas against central differences of the 64-bit
    forward, and the kernel's directional derivative against both."""
    n, b, t, h, d, rot = 2, 1, 3, 2, 16, 8
    gen = torch.Generator().manual_seed(11)
    x, w = torch.randn(n, b, t, h, d, generator=gen), 1 + 0.3 * torch.randn(n, d, generator=gen)
    cos, sin = R.tables(t, rot)
    pos = torch.arange(t)
    dy = torch.randn(n, b, t, h, d, generator=gen)
    dx, dw, _, _ = R.rope_grad(x, w, cos, sin, pos, 1e-6, False, dy)
    f = lambda xx, ww: float((R.rope(xx, ww, cos, sin, pos, 1e-6, False)[0] * dy.double()).sum())
    step = 1e-5
    for _ in range(4):
        ux, uw = torch.randn(x.shape, generator=gen).double(), torch.randn(w.shape, generator=gen).double()
        num = (f(x.double() + step * ux, w.double() + step * uw) - f(x.double() - step * ux, w.double() - step * uw)) \
            / (2 * step)
        ana = float((dx * ux).sum() + (dw * uw).sum())
        assert abs(num - ana) <= 1e-6 * (1 + abs(ana))      # step^2 of the third derivative, 64-bit cancellation
    xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    y, _ = ops.qk_norm_rope(xd, xd.detach(), wd, wd.detach(), cos.to(DEV), sin.to(DEV), pos.to(DEV))
    gx, gw = torch.autograd.grad(y, (xd, wd), dy.to(DEV))
    ux, uw = torch.randn(x.shape, generator=gen).double(), torch.randn(w.shape, generator=gen).double()
    got = float((gx.double().cpu() * ux).sum() + (gw.double().cpu() * uw).sum())
    num = (f(x.double() + step * ux, w.double() + step * uw) - f(x.double() - step * ux, w.double() - step * uw)) / (2 * step)
    assert abs(got - num) <= 1e-4 * (1 + abs(num))


def test_gradients_are_the_same_every_time():
    gen = torch.Generator().manual_seed(12)
    q, k, _ = heads(2, 4, 300, 8, 2, 128, BF16, gen)
    w = weights(2, 128, BF16, gen)
    cos, sin = (x.to(DEV) for x in R.tables(300, 128))
    pos = torch.arange(300, device=DEV)
    dyq, dyk = torch.randn(q.shape, device=DEV).to(BF16), torch.randn(k.shape, device=DEV).to(BF16)
    first = ops.qk_norm_rope_bwd(q, k, w, w, cos, sin, pos, dyq, dyk)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, ops.qk_norm_rope_bwd(q, k, w, w, cos, sin, pos, dyq, dyk)))


# ---------------------------------------------------------------------------
# Cache
# ---------------------------------------------------------------------------

def empty_cache(n, b, hk, d, tokens, page, fmt, gen, shared=False):
    """Pages of every sequence in random order; the pool holds one spare."""
    cols = -(-tokens // page)
    held = b * cols + 1
    if shared:
        table = torch.randperm(held, generator=gen)[:b * cols].view(b, cols)
    else:
        table = torch.stack([torch.randperm(held, generator=gen)[:b * cols].view(b, cols) for _ in range(n)])
    shape = (n, held, hk, page, d)
    k, v = (torch.zeros(shape, device=DEV).to(fmt) for _ in range(2))
    s = [torch.zeros(shape[:4], device=DEV) for _ in range(2)] if fmt in R.CODE_MAX else [None, None]
    return wc.WidePagedCache(k, v, table.to(torch.int32).to(DEV), *s)


CACHE = [(2, 3, 37, 2, 64, 16), (1, 1, 1, 1, 128, 64), (3, 2, 20, 4, 128, 7), (2, 2, 9, 3, 72, 24), (1, 2, 65, 1, 256, 32),
         (2, 1, 5, 2, 33, 3), (1, 3, 4, 5, 46, 1), (1, 1, 11, 2, 1, 4)]


@pytest.mark.parametrize("shape", CACHE)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("fmt", ['same', I8, E4M3])
def test_cache_write_and_read(shape, dtype, fmt):
    n, b, t, hk, d, page = shape
    fmt = dtype if fmt == 'same' else fmt
    gen = torch.Generator().manual_seed(sum(shape))
    _, k, v = heads(n, b, t, 1, hk, d, dtype, gen)
    cache = empty_cache(n, b, hk, d, t, page, fmt, gen, shared=sum(shape) % 2 == 0)
    pos = torch.stack([torch.randperm(t, generator=gen) for _ in range(b)])
    pos[torch.rand(pos.shape, generator=gen) < 0.2] = -1
    ops.cache_write(cache, k, v, pos.to(DEV))
    for out in {dtype, F32, BF16} if fmt in R.CODE_MAX else {dtype}:
        kr, vr = ops.cache_read(cache, pos.to(DEV), dtype=out)
        for got, x in ((kr, k), (vr, v)):
            want = R.held(x, fmt).to(out)
            want[(pos < 0)[None].expand(n, b, t)] = 0.0
            assert got.dtype == out and torch.equal(got.cpu(), want)          # bit for bit
    no_device_error()
    untouched = torch.ones(n, cache.pages, page, dtype=torch.bool)
    table = cache.table.cpu().long().expand(n, b, -1)
    for i in range(n):
        for j in range(b):
            p = pos[j][pos[j] >= 0]
            untouched[i, table[i, j][p // page], p % page] = False
    assert float(cache.k.float().cpu().transpose(2, 3)[untouched].abs().sum()) == 0.0


@pytest.mark.parametrize("fmt", [I8, E4M3])
def test_quantised_rows_of_zeros_tiny_and_non_finite_values(fmt):
    d = 64
    x = torch.randn(1, 1, 7, 1, d)
    x[0, 0, 1] = 0.0
    x[0, 0, 2] = 2.0 ** -60                                # under the smallest row maximum: codes 0
    x[0, 0, 3, 0, 5] = float('nan')
    x[0, 0, 4, 0, 6] = float('inf')
    x[0, 0, 5] = 3e38
    x[0, 0, 6] = torch.arange(d) * 2.0 ** -10 + 0.5         # many ties
    gen = torch.Generator().manual_seed(1)
    cache = empty_cache(1, 1, 1, d, 7, 4, fmt, gen)
    pos = torch.arange(7, device=DEV)
    ops.cache_write(cache, x.to(DEV), x.to(DEV), pos)
    k, v = (y.cpu() for y in ops.cache_read(cache, pos, dtype=F32))
    assert torch.equal(k.nan_to_num(7.0), v.nan_to_num(7.0))
    assert torch.isnan(k[0, 0, 3]).all() and torch.isnan(k[0, 0, 4]).all()
    fine = [0, 1, 2, 5, 6]
    assert torch.equal(k[:, :, fine], R.held(x[:, :, fine], fmt))
    assert float(k[0, 0, 1].abs().max()) == 0.0


def test_cache_positions_and_pages_out_of_range():
    gen = torch.Generator().manual_seed(2)
    cache = empty_cache(1, 2, 1, 64, 8, 4, BF16, gen)
    _, k, v = heads(1, 2, 1, 1, 1, 64, BF16, gen)
    before = cache.k.clone()
    ops.cache_write(cache, k, v, torch.tensor([8], device=DEV))                # past the table
    assert _native.device_error() == _native.DEV_ERR_INDEX and torch.equal(cache.k, before)
    ops.cache_write(cache, k, v, torch.tensor([2 ** 40], device=DEV))
    assert _native.device_error() == _native.DEV_ERR_INDEX and torch.equal(cache.k, before)
    cache.table[0, 1, 1] = cache.pages                                         # a page past the pool
    ops.cache_write(cache, k, v, torch.tensor([5], device=DEV))
    assert _native.device_error() == _native.DEV_ERR_INDEX
    kr, _ = ops.cache_read(cache, torch.tensor([5], device=DEV))
    assert _native.device_error() == _native.DEV_ERR_INDEX
    assert torch.equal(kr[0, 0], k[0, 0]) and float(kr[0, 1].abs().max()) == 0.0


@pytest.mark.parametrize("fmt", ['same', I8, E4M3])
@pytest.mark.parametrize("shape", [(2, 3, 1, 8, 2, 128, 128), (1, 2, 5, 3, 3, 64, 32), (2, 2, 3, 2, 1, 46, 10),
                                   (1, 4, 2, 12, 4, 80, 80)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_qk_norm_rope_write(fmt, shape, dtype):
    """The fused write: queries as the unfused call gives them, keys as the
    norm + rotation in 64 bits within one code, values bit for bit."""
    n, b, t, hq, hk, d, rot = shape
    fmt = dtype if fmt == 'same' else fmt
    gen = torch.Generator().manual_seed(sum(shape) + 5)
    q, k, v = heads(n, b, t, hq, hk, d, dtype, gen)
    qw, kw = weights(n, d, dtype, gen), weights(n, d, dtype, gen)
    cos, sin = R.tables(t + 9, rot)
    pos = torch.stack([torch.randperm(t + 9, generator=gen)[:t] for _ in range(n * b)]).view(n, b, t)
    pos[0, 0, 0] = -1
    cache = empty_cache(n, b, hk, d, t + 9, 4, fmt, gen)
    args = (qw, kw, cos.to(DEV), sin.to(DEV), pos.to(DEV))
    yq = ops.qk_norm_rope_write(q, k, v, *args, cache)
    assert torch.equal(yq, ops.qk_norm_rope(q, k, *args)[0])
    kr, vr = ops.cache_read(cache, pos.to(DEV), dtype=F32 if fmt in R.CODE_MAX else None)
    want_v = R.held(v, fmt).to(vr.dtype)
    want_v[pos < 0] = 0.0
    assert torch.equal(vr.cpu(), want_v)
    want, amp = R.rope(k, kw, cos, sin, pos, 1e-6, False)
    top = want.abs().amax(-1, keepdim=True)
    # rounding to a code: half a step (int8: top / 254; e4m3: 2^-4 of the value, or half its smallest step)
    step = {I8: top / 254, E4M3: torch.maximum(want.abs() * 2.0 ** -4, top / 448 * 2.0 ** -10)}.get(
        fmt, R.store_ulp(dtype) * want.abs() + R.tiny(dtype))
    R.assert_within(kr, want, step * (1 + 2.0 ** -6) + 2 * ROW_OPS * R.U * (amp + top))
    no_device_error()


# ---------------------------------------------------------------------------
# Attention of one new token
# ---------------------------------------------------------------------------

def fill(cache, lengths, gen, dirty=True):
    """Random values in the visible slots; what lies past a sequence's length
    (and in unused pages) is NaN: slots that no token was written to."""
    n, b = cache.n, cache.batch
    shape = cache.k.shape
    ln = lengths.long().expand(n, b)
    seen = torch.zeros(n, shape[1], shape[3], dtype=torch.bool)
    table = cache.table.cpu().long().expand(n, b, -1)
    for i in range(n):
        for j in range(b):
            p = torch.arange(int(ln[i, j]))
            seen[i, table[i, j][p // shape[3]], p % shape[3]] = True
    hide = (~seen)[:, :, None, :].expand(shape[:4]).to(DEV)
    for side, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = torch.randn(shape, generator=gen) * 1.3
        if scale is None:
            side.copy_(x)
            if dirty:
                side[hide] = float('nan')
        else:
            code, s = R.encode(x, side.dtype)
            side.copy_(code)
            scale.copy_(s)
            if dirty:
                scale[hide] = float('nan')
    return cache


# n, b, hq, hk, d, page, longest
DECODE = [
    (1, 1, 1, 1, 64, 16, 1), (2, 3, 8, 8, 64, 16, 37), (1, 2, 8, 1, 128, 64, 200), (2, 2, 16, 2, 128, 20, 301),
    (1, 3, 6, 2, 84, 7, 99), (1, 1, 12, 1, 256, 128, 515), (2, 1, 3, 3, 33, 5, 40), (1, 2, 32, 1, 96, 1, 50),
    (1, 1, 4, 4, 16, 32, 1000), (1, 2, 20, 4, 46, 33, 130), (3, 1, 2, 1, 1, 4, 9), (1, 1, 24, 1, 192, 48, 97),
    (1, 1, 40, 2, 64, 256, 2500),
]


@pytest.mark.parametrize("shape", DECODE)
@pytest.mark.parametrize("dtype,fmt", [(F32, F32), (BF16, BF16), (F16, F16), (F32, I8), (BF16, I8), (F16, I8), (F32, E4M3),
                                       (BF16, E4M3), (F16, E4M3)])
def test_decode_attention(shape, dtype, fmt):
    n, b, hq, hk, d, page, longest = shape
    gen = torch.Generator().manual_seed(sum(shape))
    lengths = torch.randint(1, longest + 1, (n, b), generator=gen, dtype=torch.int32)
    lengths[0, 0] = longest
    cache = fill(empty_cache(n, b, hk, d, longest, page, fmt, gen), lengths, gen)
    q = (torch.randn(n, b, hq, d, generator=gen) * 1.5).to(dtype).to(DEV)
    out = ops.decode_attention(q, cache, lengths.to(DEV))
    want, mag, reach = R.decode(q, cache, lengths)
    assert out.dtype == dtype and out.is_contiguous()
    R.assert_within(out, want, R.decode_bound(want, mag, reach, d, dtype))
    no_device_error()


@pytest.mark.parametrize("off", [0, 1, 2, 4])
@pytest.mark.parametrize("dtype,fmt,d", [(BF16, I8, 138), (F32, E4M3, 138), (F16, E4M3, 62), (BF16, I8, 61), (BF16, I8, 63),
                                         (F32, I8, 125), (BF16, E4M3, 127), (BF16, I8, 253), (F16, E4M3, 255), (F16, I8, 100),
                                         (BF16, E4M3, 24), (BF16, BF16, 31), (F16, F16, 127), (BF16, BF16, 255),
                                         (BF16, BF16, 68), (F32, F32, 61)])
def test_decode_rows_of_any_size_and_place(dtype, fmt, d, off):
    """Rows that start at any byte, in pools that start `off` elements into
    their storage."""
    n, b, hq, hk, page, longest = 2, 3, 12, 1, 20, 310
    gen = torch.Generator().manual_seed(d + off)
    lengths = torch.randint(1, longest + 1, (n, b), generator=gen, dtype=torch.int32)
    lengths[1, 1] = longest
    cache = fill(empty_cache(n, b, hk, d, longest, page, fmt, gen), lengths, gen)
    moved = []
    for x in (cache.k, cache.v):
        flat = torch.empty(x.numel() + 8, device=DEV, dtype=x.dtype)
        moved.append(flat[off:off + x.numel()].view(x.shape))
        moved[-1].copy_(x)
    cache = wc.WidePagedCache(*moved, cache.table, cache.k_scale, cache.v_scale)
    q = torch.randn(n, b, hq, d, generator=gen).to(dtype).to(DEV)
    out = ops.decode_attention(q, cache, lengths.to(DEV))
    want, mag, reach = R.decode(q, cache, lengths)
    R.assert_within(out, want, R.decode_bound(want, mag, reach, d, dtype))
    no_device_error()


@pytest.mark.parametrize("window", [1, 15, 16, 17, 64, 5000])
@pytest.mark.parametrize("fmt", [BF16, I8])
def test_decode_window_and_empty_sequences(window, fmt):
    n, b, hq, hk, d, page = 2, 5, 4, 2, 64, 12
    gen = torch.Generator().manual_seed(window)
    lengths = torch.tensor([[0, 1, 15, 700, 64], [33, 0, 16, 17, 699]])
    cache = fill(empty_cache(n, b, hk, d, 700, page, fmt, gen), lengths, gen)
    q = torch.randn(n, b, hq, d, generator=gen).to(BF16).to(DEV)
    out = ops.decode_attention(q, cache, lengths.to(DEV), window=window)
    want, mag, reach = R.decode(q, cache, lengths, window=window)
    R.assert_within(out, want, R.decode_bound(want, mag, reach, d, BF16))
    assert float(out[0, 0].abs().max()) == 0.0 and float(out[1, 1].abs().max()) == 0.0
    no_device_error()


@pytest.mark.parametrize("dtype,fmt", [(BF16, BF16), (F16, I8), (F32, F32)])
def test_decode_strided_queries_shared_table_and_scale(dtype, fmt):
    n, b, hq, hk, d, page = 3, 4, 6, 3, 64, 16
    gen = torch.Generator().manual_seed(21)
    lengths = torch.tensor([5, 60, 1, 33])
    cache = fill(empty_cache(n, b, hk, d, 60, page, fmt, gen, shared=True), lengths, gen)
    x = torch.randn(n, b, 2, hq + 4, d, generator=gen).to(dtype).to(DEV)
    q = x[:, :, 1, 2:2 + hq]
    out = ops.decode_attention(q, cache, lengths.to(DEV), scale=0.37)
    want, mag, reach = R.decode(q, cache, lengths, scale=0.37)
    R.assert_within(out, want, R.decode_bound(want, mag, reach, d, dtype))
    assert torch.equal(out, ops.decode_attention(q.contiguous(), cache, lengths.int().to(DEV), scale=0.37))


@pytest.mark.parametrize("dtype,fmt", [(BF16, BF16), (F16, F16), (BF16, I8), (F32, E4M3), (F32, F32)])
def test_decode_sharp_scores_and_uneven_value_scales(dtype, fmt):
    """One token far above the rest, rows of very different size, values of
    zeros, and scores so low that only the running maximum keeps them."""
    n, b, hq, hk, d, page, length = 1, 1, 8, 1, 64, 16, 400
    gen = torch.Generator().manual_seed(31)
    lengths = torch.tensor([length])
    cache = empty_cache(n, b, hk, d, length, page, fmt, gen)
    k = torch.randn(1, 1, length, 1, d, generator=gen)
    k[:, :, 123] *= 12.0
    v = torch.randn(1, 1, length, 1, d, generator=gen) * torch.logspace(
        -4, 3, length)[torch.randperm(length, generator=gen)].view(1, 1, -1, 1, 1)
    v[:, :, 50:60] = 0.0
    ops.cache_write(cache, k.to(dtype).to(DEV), v.to(dtype).to(DEV), torch.arange(length, device=DEV))
    for gain in (1.0, 20.0, 1e-3):
        q = (torch.randn(1, 1, hq, d, generator=gen) * gain).to(dtype).to(DEV)
        q[0, 0, 1] = 0.0
        out = ops.decode_attention(q, cache, lengths.to(DEV))
        want, mag, reach = R.decode(q, cache, lengths)
        R.assert_within(out, want, R.decode_bound(want, mag, reach, d, dtype))


@pytest.mark.parametrize("fmt", [F32, BF16, I8, E4M3])
def test_decode_long_cache_is_joined_and_repeats(fmt):
    dtype = BF16 if fmt in R.CODE_MAX else fmt
    n, b, hq, hk, d, page = 1, 2, 4, 1, 64, 128
    gen = torch.Generator().manual_seed(41)
    lengths = torch.tensor([20011, 3])
    cache = fill(empty_cache(n, b, hk, d, 20011, page, fmt, gen), lengths, gen)
    q = torch.randn(n, b, hq, d, generator=gen).to(dtype).to(DEV)
    out = ops.decode_attention(q, cache, lengths.to(DEV))
    want, mag, reach = R.decode(q, cache, lengths)
    R.assert_within(out, want, R.decode_bound(want, mag, reach, d, dtype))
    for _ in range(3):
        assert torch.equal(out, ops.decode_attention(q, cache, lengths.to(DEV)))


def test_decode_length_past_the_table_and_bad_pages():
    gen = torch.Generator().manual_seed(51)
    lengths = torch.tensor([30, 12])
    cache = fill(empty_cache(1, 2, 1, 64, 32, 16, BF16, gen), torch.tensor([32, 32]), gen)
    q = torch.randn(1, 2, 4, 64, generator=gen).to(BF16).to(DEV)
    ref = ops.decode_attention(q, cache, torch.tensor([32, 12], device=DEV))
    no_device_error()
    out = ops.decode_attention(q, cache, torch.tensor([77, 12], device=DEV))      # clamped to the 32 that fit
    assert _native.device_error() == _native.DEV_ERR_INDEX
    assert torch.equal(out, ref)
    cache.table[0, 0, 0] = -1                                                      # its tokens are left out
    out = ops.decode_attention(q, cache, lengths.to(DEV))
    assert _native.device_error() == _native.DEV_ERR_INDEX
    assert torch.isfinite(out).all()
    want = R.decode(q[:, :1], wc.WidePagedCache(cache.k, cache.v, cache.table[:, :1, 1:].contiguous()),
                    torch.tensor([14]))
    R.assert_within(out[:, :1], want[0], R.decode_bound(*want, 64, BF16))


def test_offsets_past_32_bits():
    """A pool whose last pages lie beyond 2^32 bytes and 2^31 elements."""
    pages, page, d = 70000, 128, 256
    k = torch.zeros(1, pages, 1, page, d, device=DEV, dtype=BF16)
    v = torch.zeros(1, pages, 1, page, d, device=DEV, dtype=BF16)
    assert k.numel() > 2 ** 31
    table = torch.tensor([[pages - 1, 0]], dtype=torch.int32, device=DEV)
    cache = wc.WidePagedCache(k, v, table)
    gen = torch.Generator().manual_seed(61)
    _, kk, vv = heads(1, 1, 200, 1, 1, d, BF16, gen)
    pos = torch.arange(200, device=DEV)
    ops.cache_write(cache, kk, vv, pos)
    kr, vr = ops.cache_read(cache, pos)
    assert torch.equal(kr, kk) and torch.equal(vr, vv)
    assert torch.equal(k[0, pages - 1, 0], kk[0, 0, :128, 0]) and torch.equal(k[0, 0, 0, :72], kk[0, 0, 128:, 0])
    q = torch.randn(1, 1, 2, d, generator=gen).to(BF16).to(DEV)
    out = ops.decode_attention(q, cache, torch.tensor([200], device=DEV))
    small = wc.WidePagedCache(torch.stack([k[:, -1], k[:, 0]], 1), torch.stack([v[:, -1], v[:, 0]], 1),
                              torch.tensor([[0, 1]], dtype=torch.int32, device=DEV))
    assert torch.equal(out, ops.decode_attention(q, small, torch.tensor([200], device=DEV)))


def test_other_streams():
    gen = torch.Generator().manual_seed(71)
    lengths = torch.tensor([900, 411])
    cache = fill(empty_cache(1, 2, 2, 128, 900, 64, BF16, gen), lengths, gen)
    q = torch.randn(1, 2, 8, 128, generator=gen).to(BF16).to(DEV)
    ln = lengths.to(DEV)
    ref = ops.decode_attention(q, cache, ln)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.decode_attention(q, cache, ln))
    torch.cuda.synchronize()
    assert all(torch.equal(ref, o) for o in outs)


def test_cuda_graph_replay_follows_new_lengths():
    gen = torch.Generator().manual_seed(81)
    lengths = torch.tensor([500, 20], dtype=torch.int32)
    cache = fill(empty_cache(1, 2, 2, 64, 500, 16, I8, gen), torch.tensor([500, 500]), gen)
    q = torch.randn(1, 2, 4, 64, generator=gen).to(BF16).to(DEV)
    ln = lengths.to(DEV)
    ops.decode_attention(q, cache, ln)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.decode_attention(q, cache, ln)
    for new in ([7, 500], [0, 1], [499, 64]):
        ln.copy_(torch.tensor(new, dtype=torch.int32))
        g.replay()
        assert torch.equal(out, ops.decode_attention(q, cache, ln))


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------

def test_refusals():
    gen = torch.Generator().manual_seed(91)
    q, k, v = heads(2, 2, 3, 4, 2, 64, BF16, gen)
    w = weights(2, 64, BF16, gen)
    cos, sin = (x.to(DEV) for x in R.tables(8, 64))
    pos = torch.arange(3, device=DEV)
    cache = empty_cache(2, 2, 2, 64, 8, 4, BF16, gen)
    with pytest.raises(TypeError, match="dtype"):
        ops.qk_norm_rope(q, k.float(), w, w, cos, sin, pos)
    with pytest.raises(ValueError, match="positions"):
        ops.qk_norm_rope(q, k, w, w, cos, sin, torch.arange(4, device=DEV))
    with pytest.raises(TypeError, match="positions"):
        ops.qk_norm_rope(q, k, w, w, cos, sin, pos.float())
    with pytest.raises(ValueError, match="weights"):
        ops.qk_norm_rope(q, k, w[:1], w, cos, sin, pos)
    with pytest.raises(ValueError, match="rotated"):
        ops.qk_norm_rope(q, k, w, w, *(torch.zeros(8, 33, device=DEV),) * 2, pos)
    with pytest.raises(ValueError, match="cos and sin"):
        ops.qk_norm_rope(q, k, w, w, cos.double(), sin.double(), pos)
    with pytest.raises(ValueError, match="dense"):
        ops.qk_norm_rope(q, k.transpose(3, 4).contiguous().transpose(3, 4), w, w, cos, sin, pos)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.qk_norm_rope(q, k, w.cpu(), w, cos, sin, pos)
    with pytest.raises(ValueError, match="256"):
        x = torch.zeros(1, 1, 1, 1, 258, device=DEV)
        ops.qk_norm_rope(x, x, x.view(1, 258), x.view(1, 258), cos, sin, pos[:1])
    with pytest.raises(ValueError, match="do not match"):
        ops.cache_write(cache, k[:1], v[:1], pos)
    with pytest.raises(TypeError, match="dtype"):
        ops.cache_write(cache, k.float(), v.float(), pos)
    with pytest.raises(TypeError, match="dtype"):
        ops.cache_read(cache, pos, dtype=F16)
    with pytest.raises(ValueError, match="query heads"):
        ops.decode_attention(torch.zeros(2, 2, 3, 64, device=DEV, dtype=BF16), cache, pos[:2])
    with pytest.raises(ValueError, match="lengths"):
        ops.decode_attention(q[:, :, 0], cache, pos)
    with pytest.raises(ValueError, match="window"):
        ops.decode_attention(q[:, :, 0], cache, pos[:2], window=-1)
    with pytest.raises(ValueError, match="scales"):
        wc.WidePagedCache(cache.k.to(I8), cache.v.to(I8), cache.table)
    with pytest.raises(ValueError, match="int32"):
        wc.WidePagedCache(cache.k, cache.v, cache.table.long())
    with pytest.raises(ValueError, match="contiguous"):
        wc.WidePagedCache(cache.k.transpose(2, 3), cache.v.transpose(2, 3), cache.table)
    no_device_error()


@pytest.mark.grad
def test_cache_paths_refuse_gradients():
    gen = torch.Generator().manual_seed(92)
    q, k, v = heads(1, 1, 1, 2, 1, 64, BF16, gen)
    cache = empty_cache(1, 1, 1, 64, 8, 4, BF16, gen)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.cache_write(cache, k.detach().requires_grad_(True), v, torch.zeros(1, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="gradient"):
        ops.decode_attention(q[:, :, 0].detach().requires_grad_(True), cache, torch.ones(1, dtype=torch.int32, device=DEV))


def test_empty_calls():
    w = torch.ones(2, 64, device=DEV)
    cos, sin = (x.to(DEV) for x in R.tables(4, 64))
    x = torch.zeros(2, 3, 0, 2, 64, device=DEV)
    pos = torch.zeros(0, dtype=torch.int64, device=DEV)
    yq, yk = ops.qk_norm_rope(x, x, w, w, cos, sin, pos)
    assert yq.shape == x.shape
    grads = ops.qk_norm_rope_bwd(x, x, w, w, cos, sin, pos, yq, yk)
    assert grads[0].shape == x.shape and float(grads[2].abs().sum()) == 0.0
    cache = wc.WidePagedCache.allocate(2, 3, 2, 64, max_len=16, page_size=8, dtype=F32)
    ops.cache_write(cache, x, x, pos)
    assert ops.cache_read(cache, pos)[0].shape == x.shape
    none = wc.WidePagedCache.allocate(2, 0, 2, 64, max_len=16, page_size=8, dtype=F32)
    assert ops.decode_attention(torch.zeros(2, 0, 4, 64, device=DEV), none,
                                torch.zeros(0, dtype=torch.int32, device=DEV)).shape == (2, 0, 4, 64)
    no_room = wc.WidePagedCache.allocate(1, 2, 2, 64, max_len=0, page_size=8, dtype=F32)
    out = ops.decode_attention(torch.ones(1, 2, 4, 64, device=DEV), no_room,
                               torch.zeros(2, dtype=torch.int32, device=DEV))
    assert float(out.abs().max()) == 0.0
    no_device_error()
