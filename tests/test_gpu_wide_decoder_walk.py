"""Attention of one new token where a block of the kernel takes many steps:
its ring is used again and again, the running maximum moves between its steps,
it crosses from one segment into the next, and a segment lies in several
blocks. Against the definition in 64 bits (decoder_ref.decode, here on the
device for its speed)."""
import math

import pytest
import torch

import decoder_ref as R
import wide_compiler as wc
from gpu_util import no_device_error
from wide_compiler import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
I8, E4M3 = torch.int8, torch.float8_e4m3fn
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (F32, I8), (BF16, I8), (F16, I8), (F32, E4M3), (BF16, E4M3), (F16, E4M3)]


def steps_of_a_block(cache, lengths, group, window=0):
    """Steps that each block takes at least, by the entry's own division (the
    last block may have fewer)."""
    d, page = cache.head_dim, cache.page_size
    size = cache.k.element_size()
    bytes_ = (64 if d <= 64 else 128 if d <= 128 else 256) * size
    step = 64 * (1 if bytes_ >= 512 else 2 if bytes_ == 256 else 256 // bytes_)
    nt = 2 if group > 8 and d <= 128 and cache.k.dtype != F32 else 1
    tiles = -(-group // (8 * nt))
    places = 1 if bytes_ > 512 else 2 if bytes_ >= 256 or nt == 2 or d > 128 else 3
    blocks = places * torch.cuda.get_device_properties(0).multi_processor_count
    ln = lengths.long().expand(cache.n, cache.batch)
    seen = ln.clamp(max=window) if window else ln
    return int(((seen + step - 1) // step).clamp(min=1).sum()) * cache.kv_heads * tiles / blocks


def encode(x, fmt):
    """decoder_ref.encode on the device."""
    if fmt not in R.CODE_MAX:
        return x.to(fmt), None
    top = x.abs().amax(-1).clamp(min=2.0 ** -40)
    scale = top / torch.full_like(top, R.CODE_MAX[fmt])
    y = x / scale.unsqueeze(-1)
    return (torch.round(y) if fmt == I8 else y).to(fmt), scale


def cache_of(n, b, hk, d, page, fmt, lengths, gen, wave):
    """Pages in random order; keys that grow and shrink along the sequence (so
    that the largest score moves), NaN in every slot past a length."""
    cols = -(-max(int(lengths.max()), 1) // page)
    held = b * cols + 1
    table = torch.rand(n, held, device=DEV, generator=gen).argsort(1)[:, :b * cols].view(n, b, cols).to(torch.int32)
    shape = (n, held, hk, page, d)
    place = torch.zeros(n, held, page, device=DEV, dtype=torch.long)      # token held there
    seen = torch.zeros(n, held, page, device=DEV, dtype=torch.bool)
    at = torch.arange(n, device=DEV)[:, None, None]
    tok = torch.arange(cols * page, device=DEV).view(cols, page)
    place[at, table.long()] = tok
    seen[at, table.long()] = tok < lengths.long().expand(n, b)[:, :, None, None]
    sides = []
    for key in (True, False):
        x = torch.randn(shape, device=DEV, generator=gen)
        if key:
            x *= 1 + wave * torch.sin(place / 97.0)[:, :, None, :, None]
        sides.append(encode(x, fmt))
    for code, scale in sides:
        (code if scale is None else scale)[~seen[:, :, None, :].expand(shape[:4])] = float('nan')
    (k, ks), (v, vs) = sides
    return wc.WidePagedCache(k, v, table, ks, vs)


def decode_on_device(q, cache, lengths, scale=None, window=0):
    """decoder_ref.decode in 64 bits on the device, a sequence at a time."""
    n, b, hq, d = q.shape
    hk, page = cache.kv_heads, cache.page_size
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(q.shape, device=DEV, dtype=torch.float64)
    mag, reach = torch.zeros_like(out), torch.zeros(n, b, hq, device=DEV, dtype=torch.float64)
    table = cache.table.long().expand(n, b, -1)
    ln = lengths.long().expand(n, b).tolist()
    bits = lambda x: x.view(torch.uint8) if x.dtype == E4M3 else x
    for i in range(n):
        for j in range(b):
            hi = ln[i][j]
            lo = max(0, hi - window) if window else 0
            if hi <= lo:
                continue
            p = torch.arange(lo, hi, device=DEV)
            at, off = table[i, j][p // page], p % page
            side = []
            for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
                y = bits(x[i])[at, :, off].view(x.dtype).double()                   # [L, Hk, D]
                side.append(y if s is None else y * s[i][at, :, off].double().unsqueeze(-1))
            k, v = side
            qq = q[i, j].double().view(hk, hq // hk, d)
            z = scale * torch.einsum('hgd,lhd->hgl', qq, k)
            w = torch.softmax(z, -1)
            out[i, j] = torch.einsum('hgl,lhd->hgd', w, v).reshape(hq, d)
            mag[i, j] = torch.einsum('hgl,lhd->hgd', w, v.abs()).reshape(hq, d)
            reach[i, j] = (scale * torch.einsum('hgd,lhd->hgl', qq.abs(), k.abs())).amax(-1).reshape(hq)
    return out.cpu(), mag.cpu(), reach.cpu()


def check(q, cache, lengths, **kw):
    out = ops.decode_attention(q, cache, lengths, **kw)
    want, mag, reach = decode_on_device(q, cache, lengths, **kw)
    R.assert_within(out, want, R.decode_bound(want, mag, reach, q.shape[-1], q.dtype))
    assert torch.equal(out, ops.decode_attention(q, cache, lengths, **kw))          # the same every time
    no_device_error()
    return out


# head size and query heads of a key head: every tile width, one and two head
# tiles, rows that fill the tiles, rows of 16 bytes' multiples and others
@pytest.mark.parametrize("d,group", [(64, 1), (64, 12), (84, 3), (128, 4), (128, 16), (80, 9), (138, 2), (192, 8), (256, 1)])
@pytest.mark.parametrize("dtype,fmt", TYPES)
def test_blocks_of_many_steps(dtype, fmt, d, group):
    n, b, hk, page = 2, 32, 3, 36
    gen = torch.Generator(device=DEV).manual_seed(d + group)
    lengths = torch.randint(1, 5000, (n, b), device=DEV, generator=gen, dtype=torch.int32)
    lengths[0, 3:6] = 0                                # borders with nothing between them
    lengths[1, 7] = 1
    cache = cache_of(n, b, hk, d, page, fmt, lengths, gen, wave=0.8)
    q = (torch.randn(n, b, hk * group, d, device=DEV, generator=gen) * 1.5).to(dtype)
    assert steps_of_a_block(cache, lengths, group) > 2
    out = check(q, cache, lengths)
    assert float(out[0, 3:6].abs().max()) == 0.0


@pytest.mark.parametrize("dtype,fmt", TYPES)
def test_one_segment_over_many_blocks_of_many_steps(dtype, fmt):
    """Three long segments: each lies in many blocks, each block takes many
    steps, and a border lies inside one."""
    n, b, hk, d, page = 1, 3, 1, 64, 128
    gen = torch.Generator(device=DEV).manual_seed(5)
    lengths = torch.tensor([[190001, 63, 300007]], device=DEV, dtype=torch.int32)
    cache = cache_of(n, b, hk, d, page, fmt, lengths, gen, wave=0.5)
    q = torch.randn(n, b, 4, d, device=DEV, generator=gen).to(dtype)
    assert steps_of_a_block(cache, lengths, 4) > 3
    check(q, cache, lengths)


@pytest.mark.parametrize("off", [1, 2])
@pytest.mark.parametrize("dtype,fmt,d,group", [(BF16, I8, 61, 3), (F16, E4M3, 63, 9), (F32, I8, 125, 2), (BF16, E4M3, 127, 12),
                                               (F32, E4M3, 250, 1), (BF16, BF16, 31, 2), (F16, F16, 127, 10),
                                               (BF16, BF16, 66, 1), (F32, F32, 61, 4), (F32, F32, 129, 1)])
def test_rows_of_any_place_in_blocks_of_many_steps(dtype, fmt, d, group, off):
    """Rows that start at any byte, in pools that start `off` elements into
    their storage."""
    n, b, hk, page = 2, 32, 3, 20
    gen = torch.Generator(device=DEV).manual_seed(d + off)
    lengths = torch.randint(0, 4000, (n, b), device=DEV, generator=gen, dtype=torch.int32)
    cache = cache_of(n, b, hk, d, page, fmt, lengths, gen, wave=0.8)
    moved = []
    for x in (cache.k, cache.v):
        flat = torch.empty(x.numel() + 8, device=DEV, dtype=x.dtype)
        moved.append(flat[off:off + x.numel()].view(x.shape))
        moved[-1].copy_(x)
    cache = wc.WidePagedCache(*moved, cache.table, cache.k_scale, cache.v_scale)
    q = torch.randn(n, b, hk * group, d, device=DEV, generator=gen).to(dtype)
    assert steps_of_a_block(cache, lengths, group) > 1.5
    check(q, cache, lengths)


@pytest.mark.parametrize("dtype,fmt", [(F32, F32), (BF16, BF16), (F16, I8), (F32, E4M3)])
def test_windows_over_blocks_of_many_steps(dtype, fmt):
    n, b, hk, d, page, window = 2, 40, 4, 64, 24, 1900
    gen = torch.Generator(device=DEV).manual_seed(9)
    lengths = torch.randint(0, 4000, (n, b), device=DEV, generator=gen, dtype=torch.int32)
    cache = cache_of(n, b, hk, d, page, fmt, lengths, gen, wave=0.8)
    q = torch.randn(n, b, hk * 2, d, device=DEV, generator=gen).to(dtype)
    assert steps_of_a_block(cache, lengths, 2, window) > 1.5
    check(q, cache, lengths, window=window)


@pytest.mark.parametrize("dtype,fmt", [(F32, F32), (BF16, BF16), (F16, I8), (F32, E4M3)])
@pytest.mark.parametrize("n,b,longest", [(3, 1500, 700), (2, 700, 60)])
def test_whole_segments_in_turn(dtype, fmt, n, b, longest):
    """More than 4096 sequences, and many of one step each: every block takes
    several whole segments."""
    hk, d, page = 1 if longest > 60 else 2, 64, 20
    gen = torch.Generator(device=DEV).manual_seed(longest)
    lengths = torch.randint(0, longest + 1, (n, b), device=DEV, generator=gen, dtype=torch.int32)
    cache = cache_of(n, b, hk, d, page, fmt, lengths, gen, wave=0.8)
    q = torch.randn(n, b, hk * 2, d, device=DEV, generator=gen).to(dtype)
    assert n * b * hk > 3 * 3 * torch.cuda.get_device_properties(0).multi_processor_count
    check(q, cache, lengths)


@pytest.mark.parametrize("dtype,fmt", [(F16, F16), (BF16, BF16), (F16, I8), (F16, E4M3), (F32, F32), (F32, I8)])
def test_long_sums_of_one_sign_are_not_biased(dtype, fmt):
    """131072 values of one sign summed by one block: sums that round towards
    zero would all lose the same way. The mean of the signed relative errors
    keeps that and averages out the results' own rounding (uniform, at most
    2^-p: 2^-11 or 2^-8 / sqrt(3 * 16384) here, 2.2e-6 or 1.8e-5, and more than
    three times that allowed); the weights' pieces allow 2^-16 themselves."""
    n, b, hk, d, page, held, length = 16, 4, 8, 128, 128, 32, 131072
    gen = torch.Generator(device=DEV).manual_seed(3)
    base = 1 + torch.rand(n, 1, hk, 1, d, device=DEV, generator=gen)
    v = base * (0.9 + 0.2 * torch.rand(n, held, hk, page, d, device=DEV, generator=gen))
    k = 0.3 * torch.randn(n, held, hk, page, d, device=DEV, generator=gen)
    table = torch.randint(0, held, (n, b, length // page), device=DEV, generator=gen, dtype=torch.int32)
    (k, ks), (v, vs) = encode(k, fmt), encode(v, fmt)
    cache = wc.WidePagedCache(k, v, table, ks, vs)
    q = torch.randn(n, b, hk, d, device=DEV, generator=gen).to(dtype)
    lengths = torch.full((n, b), length, device=DEV, dtype=torch.int32)
    assert steps_of_a_block(cache, lengths, 1) > 500
    out = ops.decode_attention(q, cache, lengths)
    wide = lambda x, s: x.double() if s is None else x.double() * s.double().unsqueeze(-1)
    want = torch.empty(q.shape, device=DEV, dtype=torch.float64)
    for i in range(n):
        kk, vv = wide(k[i], None if ks is None else ks[i]), wide(v[i], None if vs is None else vs[i])
        times = torch.stack([torch.bincount(table[i, j].long(), minlength=held) for j in range(b)]).double()
        w = torch.exp(torch.einsum('bhd,phtd->bhpt', q[i].double(), kk) / math.sqrt(d)) * times[:, None, :, None]
        want[i] = torch.einsum('bhpt,phtd->bhd', w, vv) / w.sum((2, 3)).unsqueeze(-1)
    err = (out.double() - want) / want
    assert abs(float(err.mean())) <= {F32: 2.0 ** -20, F16: 2.0 ** -16, BF16: 2.0 ** -14}[dtype]
    # the rounding of one result, and what decode_bound allows the weights
    assert float(err.abs().max()) <= R.store_ulp(dtype) + 2 * (2.0 ** -20 + (2.0 ** -20 if dtype == F32 else 2.0 ** -16)
                                                               + (d + 8) * R.U * 4)


@pytest.mark.parametrize("d,group", [(64, 2), (128, 1), (128, 12), (256, 2)])
@pytest.mark.parametrize("dtype,fmt", [(BF16, BF16), (F16, F16), (BF16, I8), (F16, E4M3), (F32, F32)])
def test_totals_of_chains_follow_the_maximum(dtype, fmt, d, group):
    """Whole sequences of several thousand tokens in one block, whose keys grow
    (or shrink) towards the end, so that sums of many steps ago are rescaled."""
    n, b, hk, page, held = 4, 16, 8, 100, 40
    gen = torch.Generator(device=DEV).manual_seed(d + group)
    gain = torch.linspace(0.1, 2.5, held, device=DEV).view(1, held, 1, 1, 1)
    k = gain * torch.randn(n, held, hk, page, d, device=DEV, generator=gen)
    v = torch.randn(n, held, hk, page, d, device=DEV, generator=gen)
    (k, ks), (v, vs) = encode(k, fmt), encode(v, fmt)
    lengths = torch.randint(9000, 14000, (n, b), device=DEV, generator=gen, dtype=torch.int32)
    cols = 14000 // page
    table = torch.randint(0, held, (n, b, cols), device=DEV, generator=gen, dtype=torch.int32).sort(-1).values
    table[:, ::2] = table[:, ::2].flip(-1)
    cache = wc.WidePagedCache(k, v, table, ks, vs)
    q = torch.randn(n, b, hk * group, d, device=DEV, generator=gen).to(dtype)
    assert steps_of_a_block(cache, lengths, group) > 40
    check(q, cache, lengths)


@pytest.mark.parametrize("dtype,fmt", [(BF16, BF16), (F16, E4M3), (F32, I8)])
def test_long_segments_in_turn(dtype, fmt):
    """More than 4096 sequences, some of them longer than one chain of sums."""
    n, b, hk, d, page, held, longest = 3, 1500, 1, 64, 100, 64, 6000
    gen = torch.Generator(device=DEV).manual_seed(13)
    (k, ks), (v, vs) = (encode(torch.randn(n, held, hk, page, d, device=DEV, generator=gen), fmt) for _ in range(2))
    table = torch.randint(0, held, (n, b, longest // page), device=DEV, generator=gen, dtype=torch.int32)
    lengths = torch.randint(0, longest + 1, (n, b), device=DEV, generator=gen, dtype=torch.int32)
    cache = wc.WidePagedCache(k, v, table, ks, vs)
    q = torch.randn(n, b, hk * 2, d, device=DEV, generator=gen).to(dtype)
    check(q, cache, lengths)
