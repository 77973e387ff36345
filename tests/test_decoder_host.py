"""Host-side checks of the decoder-attention operators (no GPU): the C entries
refuse bad arguments before any CUDA call, WidePagedCache checks its tensors,
the torch formulations and fake implementations agree with the 64-bit
formulas, and the index arithmetic that the kernels rely on."""
import struct

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import decoder_ref as R
import wide_compiler as wc
from wide_compiler import _autograd as AG
from wide_compiler import _native as N

P = 16                               # a stand-in pointer: never dereferenced on these paths


def rows(n=2, b=2, t=3, hq=4, hk=2, d=64, rot=64, table=8):
    g = [n, b, t, hq, hk, d, rot, table]
    for h in (hq, hk, hk):
        g += [b * t * h * d, t * h * d, h * d, d]
    return struct.pack('=23q', *g, 0, t, 1)


def cache(pages=4, page=4, cols=2, tn=4, tb=2):
    return struct.pack('=5q', pages, page, cols, tn, tb)


def decode(n=2, b=2, hq=4, hk=2, d=64):
    return struct.pack('=10q', n, b, hq, hk, d, b * hq * d, hq * d, d, b, 1)


def test_row_entries_refuse_bad_arguments():
    lib = N.load()
    fwd = lambda g, dtype=N.BF16, q=P: lib.widek_qk_norm_rope_fwd(q, P, P, P, P, P, P, P, P, g, 1e-6, 0, 0, dtype, None)
    assert fwd(rows(n=-1)) == N.WIDEK_ERR_INVALID and "out of range" in N.last_error()
    assert fwd(rows(d=258)) == N.WIDEK_ERR_UNSUPPORTED and "256" in N.last_error()
    assert fwd(rows(rot=7)) == N.WIDEK_ERR_INVALID
    assert fwd(rows(rot=66)) == N.WIDEK_ERR_INVALID
    assert fwd(rows(hq=0)) == N.WIDEK_ERR_INVALID
    assert fwd(rows(), q=None) == N.WIDEK_ERR_INVALID and "null" in N.last_error()
    assert fwd(rows(), dtype=7) == N.WIDEK_ERR_INVALID and "dtype" in N.last_error()
    assert fwd(rows(b=1 << 20, t=1 << 20)) == N.WIDEK_ERR_INVALID and "2^31" in N.last_error()
    assert fwd(None) == N.WIDEK_ERR_INVALID
    assert fwd(rows(t=0), q=None) == N.WIDEK_OK
    assert lib.widek_qk_norm_rope_bwd_workspace(rows(d=300)) == -1
    ws = lib.widek_qk_norm_rope_bwd_workspace(rows())
    assert ws > 0
    bwd = lambda size: lib.widek_qk_norm_rope_bwd(P, P, P, P, P, P, P, P, P, P, P, P, P, rows(), 1e-6, 0, 0, N.BF16, P, size,
                                                  None)
    assert bwd(ws - 1) == N.WIDEK_ERR_INVALID and "workspace" in N.last_error()


def test_cache_entries_refuse_bad_arguments():
    lib = N.load()
    write = lambda c, fmt=N.I8, dtype=N.BF16, ks=P: lib.widek_cache_write_fwd(P, P, P, P, P, ks, P, P, rows(), c, 0, fmt,
                                                                              dtype, None)
    read = lambda c, fmt=N.I8: lib.widek_cache_read_fwd(P, P, P, P, P, P, P, P, rows(), c, 0, fmt, N.BF16, None)
    for f in (write, read):
        assert f(cache(page=0)) == N.WIDEK_ERR_INVALID
        assert f(cache(pages=-1)) == N.WIDEK_ERR_INVALID
        assert f(cache(pages=1 << 30, page=4)) == N.WIDEK_ERR_INVALID and "2^31" in N.last_error()
        assert f(cache(cols=1 << 30)) == N.WIDEK_ERR_INVALID and "2^31" in N.last_error()
        assert f(cache(), fmt=N.F32) == N.WIDEK_ERR_INVALID and "type" in N.last_error()
        assert f(cache(), fmt=9) == N.WIDEK_ERR_INVALID
        assert f(None) == N.WIDEK_ERR_INVALID
    assert write(cache(), ks=None) == N.WIDEK_ERR_INVALID and "null" in N.last_error()
    assert write(cache(), fmt=9, dtype=9) == N.WIDEK_ERR_INVALID


def test_decode_entry_refuses_bad_arguments():
    lib = N.load()
    size = lambda g=decode(), c=cache(), w=0, fmt=N.BF16: lib.widek_decode_attention_workspace(g, c, w, fmt)
    call = lambda g=decode(), c=cache(), w=0, fmt=N.BF16, dtype=N.BF16, q=P, ws=P, n=1 << 30: \
        lib.widek_decode_attention_fwd(q, P, P, P, P, P, P, P, g, c, 0.1, w, 0, fmt, dtype, ws, n, None)
    assert size() >= 0
    for kw in (dict(g=decode(hq=3)), dict(g=decode(hk=0)), dict(g=decode(n=-1)), dict(g=decode(n=1 << 20, b=1 << 20)),
               dict(w=-1), dict(fmt=9), dict(g=None), dict(c=None)):
        assert size(**kw) == -1, kw
        assert call(**kw) == N.WIDEK_ERR_INVALID, kw
    assert size(g=decode(d=257)) == -1 and call(g=decode(d=257)) == N.WIDEK_ERR_UNSUPPORTED
    assert call(dtype=9) == N.WIDEK_ERR_INVALID and "dtype" in N.last_error()
    assert call(dtype=N.F16) == N.WIDEK_ERR_INVALID and "type" in N.last_error()
    assert call(q=None) == N.WIDEK_ERR_INVALID and "null" in N.last_error()
    assert call(g=decode(b=0), q=None) == N.WIDEK_OK
    long = cache(pages=4000, page=64, cols=4000)
    need = size(c=long)
    assert need > 0
    assert call(c=long, n=need - 1) == N.WIDEK_ERR_INVALID and "workspace" in N.last_error()
    assert call(c=long, ws=None) == N.WIDEK_ERR_INVALID


def test_paged_cache_checks_its_tensors():
    k = torch.zeros(2, 5, 3, 4, 8)
    t = torch.zeros(6, 2, dtype=torch.int32)
    c = wc.WidePagedCache(k, k.clone(), t)
    assert (c.n, c.batch, c.kv_heads, c.head_dim, c.pages, c.page_size, c.max_len) == (2, 6, 3, 8, 5, 4, 8)
    assert not c.quantized and struct.unpack('=5q', c.geom) == (5, 4, 2, 0, 2)
    s = torch.zeros(2, 5, 3, 4)
    q = wc.WidePagedCache(k.to(torch.int8), k.to(torch.int8), t.expand(2, 6, 2), s, s.clone())
    assert q.quantized and struct.unpack('=5q', q.geom) == (5, 4, 2, 0, 2)
    assert "int8" in repr(q)
    for bad in ((k, k[:1], t), (k, k.double(), t), (k[0], k[0], t), (k.transpose(1, 2), k.transpose(1, 2), t),
                (k, k, t.long()), (k, k, t[0]), (k, k, t.expand(3, 6, 2)), (k, k, t.t()), (k, k, t, s, s),
                (k.to(torch.int8), k.to(torch.int8), t), (k.to(torch.int8), k.to(torch.int8), t, s, s.double()),
                (k.to(torch.int8), k.to(torch.int8), t, s, s[:1])):
        with pytest.raises(ValueError):
            wc.WidePagedCache(*bad)
    with pytest.raises(TypeError):
        wc.WidePagedCache(k.double(), k.double(), t)
    a = wc.WidePagedCache.allocate(2, 3, 4, 16, max_len=33, page_size=8, dtype=torch.float8_e4m3fn, device='cpu')
    assert a.max_len == 40 and a.table.flatten().tolist() == list(range(15)) and a.k_scale.shape == (2, 15, 4, 8)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [0, 6, 16])
def test_torch_formulation_matches_the_64_bit_formulas(rot, interleaved):
    gen = torch.Generator().manual_seed(rot)
    n, b, t, d = 2, 3, 4, 16
    x = torch.randn(n, b, t, 2, d, generator=gen).requires_grad_(True)
    w = (1 + 0.2 * torch.randn(n, d, generator=gen)).requires_grad_(True)
    cos, sin = R.tables(9, rot)
    pos = torch.randint(-1, 9, (b, t), generator=gen)
    y, _ = AG.qk_norm_rope_t(x, x.detach(), w, w.detach(), cos, sin, pos, 1e-6, interleaved)
    want, amp = R.rope(x.detach(), w.detach(), cos, sin, pos, 1e-6, interleaved)
    R.assert_within(y.detach(), want, 24 * R.U * amp)
    dy = torch.randn(y.shape, generator=gen)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    dx, dw, dx_amp, dw_amp = R.rope_grad(x.detach(), w.detach(), cos, sin, pos, 1e-6, interleaved, dy)
    R.assert_within(gx, dx, 48 * R.U * dx_amp)
    R.assert_within(gw, dw, (24 + b * t * 2) * R.U * dw_amp)


def test_fake_implementations():
    with FakeTensorMode():
        t = lambda *s, dt=torch.bfloat16: torch.empty(*s, device='cuda', dtype=dt)
        q, k, w = t(2, 3, 4, 6, 32), t(2, 3, 4, 2, 32), t(2, 32)
        cos = t(9, 16, dt=torch.float32)
        pos = torch.empty(3, 4, device='cuda', dtype=torch.int32)
        ops = torch.ops.widek
        got = ops.qk_norm_rope(q, k, w, w, cos, cos, pos, 1e-6, False)
        assert [tuple(x.shape) for x in got] == [tuple(q.shape), tuple(k.shape)]
        want = AG.qk_norm_rope_t(q, k, w, w, cos, cos, pos, 1e-6, False)
        assert [(x.shape, x.dtype) for x in got] == [(x.shape, x.dtype) for x in want]
        pages = t(2, 9, 2, 16, 32, dt=torch.int8)
        scale = t(2, 9, 2, 16, dt=torch.float32)
        table = torch.empty(3, 3, device='cuda', dtype=torch.int32)
        held = (pages, pages.clone(), table, scale, scale.clone())
        assert ops.qk_norm_rope_write(q, k, k, w, w, cos, cos, pos, held[0], held[1], table, held[3], held[4], 1e-6,
                                      False).shape == q.shape
        ops.cache_write(*held, k, k, pos)
        kr, vr = ops.cache_read(*held, pos, torch.float16)
        assert kr.shape == vr.shape == k.shape and kr.dtype == torch.float16
        assert ops.cache_read(*held, pos, None)[0].dtype == torch.bfloat16
        ln = torch.empty(3, device='cuda', dtype=torch.int32)
        out = ops.decode_attention(q[:, :, 0], *held, ln, 0.1, 0)
        assert out.shape == (2, 3, 6, 32) and out.dtype == torch.bfloat16


def test_quotient_by_multiplication_over_the_whole_range():
    """The kernels' division by a fixed divisor: q = (hi(x m) + x) >> s for
    every dividend below 2^31 (exact at the ends, at multiples and beside
    them, and at random)."""
    gen = torch.Generator().manual_seed(0)
    divisors = [1, 2, 3, 5, 7, 16, 24, 64, 100, 127, 128, 1000, 12345, 65535, 65536, 1 << 20, (1 << 30) + 1, (1 << 31) - 1]
    for d in divisors:
        s = 0
        while s < 32 and (1 << s) < d:
            s += 1
        m = ((((1 << s) - d) << 32) // d + 1) & 0xffffffff
        xs = {0, 1, d - 1, d, d + 1, (1 << 31) - 1, (1 << 31) - 2}
        xs |= {k * d + e for k in torch.randint(0, max(((1 << 31) - 1) // d, 1), (200,), generator=gen).tolist()
               for e in (-1, 0, 1)}
        xs |= set(torch.randint(0, (1 << 31) - 1, (200,), generator=gen).tolist())
        for x in xs:
            if 0 <= x < (1 << 31):
                assert (((x * m) >> 32) + x) >> s == x // d, (x, d)


def test_decoder_layer_checks_and_fusing():
    with pytest.raises(ValueError):
        wc.WideDecoderAttention(2, 64, 4, 3)
    with pytest.raises(ValueError):
        wc.WideDecoderAttention(2, 65, 4)
    ones = [wc.WideDecoderAttention(1, 64, 4, 2, bias=True) for _ in range(3)]
    wide = wc.WideDecoderAttention.from_modules(ones)
    assert wide.n == 3 and torch.equal(wide.qkv_weight[1], ones[1].qkv_weight[0])
    assert torch.equal(wide.out_bias[2], ones[2].out_bias[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        wide(torch.zeros(3, 1, 2, 64))
