"""64-bit formulas of the decoder-attention operators, written from their
definitions (loops over tokens and heads where that is plainest), and the
error bounds the tests hold the kernels to.

Bounds. One fp32 operation rounds by at most U = 2^-24 relative to its result;
a result stored in a type with p significand bits by 2^-p (bf16: 2^-9, f16:
2^-12, plus half its smallest subnormal).
"""
import math

import torch

U = 2.0 ** -24
CODE_MAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def store_ulp(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}[dtype]


def tables(rows, rot, base=10000.0):
    i = torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1)
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * base ** (-i)[None]
    return torch.cos(ang).float(), torch.sin(ang).float()


def pairs(rot, interleaved):
    return [(2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2) for i in range(rot // 2)]


def expand_index(p, shape):
    return p.long().expand(*shape)


def rope(x, w, cos, sin, positions, eps, interleaved):
    """y and the magnitude |u_a| + |u_b| that its rounding is relative to."""
    x, w = x.double().cpu(), w.double().cpu()
    n, b, t, h, d = x.shape
    pos = expand_index(positions.cpu(), (n, b, t))
    u = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.view(n, 1, 1, 1, d)
    y, amp = u.clone(), u.abs()
    c, s = cos.double().cpu()[pos.clamp(min=0)], sin.double().cpu()[pos.clamp(min=0)]      # [N, B, T, R/2]
    for i, (a, bb) in enumerate(pairs(2 * cos.shape[1], interleaved)):
        ci, si = c[..., i, None], s[..., i, None]
        y[..., a] = u[..., a] * ci - u[..., bb] * si
        y[..., bb] = u[..., bb] * ci + u[..., a] * si
        amp[..., a] = amp[..., bb] = u[..., a].abs() + u[..., bb].abs()
    pad = (pos < 0)[..., None, None].expand_as(y)
    return y.masked_fill(pad, 0.0), amp.masked_fill(pad, 0.0)


def rope_grad(x, w, cos, sin, positions, eps, interleaved, dy):
    """(dx, dw) by the formulas, and the magnitudes their rounding is relative
    to."""
    x, w, dy = x.double().cpu(), w.double().cpu(), dy.double().cpu()
    n, b, t, h, d = x.shape
    pos = expand_index(positions.cpu(), (n, b, t))
    pad = (pos < 0)[..., None, None].expand_as(x)
    x, dy = x.masked_fill(pad, 1.0), dy.masked_fill(pad, 0.0)
    du, amp = dy.clone(), dy.abs()
    c, s = cos.double().cpu()[pos.clamp(min=0)], sin.double().cpu()[pos.clamp(min=0)]
    for i, (a, bb) in enumerate(pairs(2 * cos.shape[1], interleaved)):
        ci, si = c[..., i, None], s[..., i, None]
        du[..., a] = dy[..., a] * ci + dy[..., bb] * si
        du[..., bb] = dy[..., bb] * ci - dy[..., a] * si
        amp[..., a] = amp[..., bb] = dy[..., a].abs() + dy[..., bb].abs()
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    wv = w.view(n, 1, 1, 1, d)
    g, gamp = du * wv, amp * wv.abs()
    dx = r * (g - x * r * r * (g * x).mean(-1, keepdim=True))
    dx_amp = r * (gamp + x.abs() * r * r * (gamp * x.abs()).mean(-1, keepdim=True))
    return dx, (du * x * r).sum((1, 2, 3)), dx_amp, (amp * x.abs() * r).sum((1, 2, 3))


def encode(x, dtype):
    """Codes and scales of 8-bit rows by the written definition, in fp32: the
    division is rounded once, then the code half to even."""
    x = x.float().cpu()
    top = x.abs().amax(-1).clamp(min=2.0 ** -40)
    scale = top / torch.full_like(top, CODE_MAX[dtype])
    y = x / scale.unsqueeze(-1)
    return (torch.round(y) if dtype == torch.int8 else y).to(dtype), scale


def held(x, dtype):
    """The fp32 values that a cache of ``dtype`` holds for rows x."""
    if dtype not in CODE_MAX:
        return x.to(dtype).float().cpu()
    code, scale = encode(x, dtype)
    return code.float() * scale.unsqueeze(-1)


def cache_value(pages, scale):
    y = pages.cpu().to(torch.float32).double()
    return y if scale is None else y * scale.double().cpu().unsqueeze(-1)


def decode(q, cache, lengths, scale=None, window=0):
    """out and the magnitudes of the error bound: sum p |v| per channel and the
    largest scale * sum |q k| of the head."""
    q = q.double().cpu()
    n, b, hq, d = q.shape
    hk, page = cache.kv_heads, cache.page_size
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    k, v = cache_value(cache.k, cache.k_scale), cache_value(cache.v, cache.v_scale)
    table = cache.table.cpu().long().expand(n, b, -1)
    ln = lengths.cpu().long().expand(n, b)
    out, mag, reach = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(n, b, hq, dtype=torch.float64)
    for i in range(n):
        for j in range(b):
            hi = int(ln[i, j])
            lo = max(0, hi - window) if window else 0
            if hi <= lo:
                continue
            p = torch.arange(lo, hi)
            at, off = table[i, j][p // page], p % page
            kk, vv = k[i, at, :, off], v[i, at, :, off]                     # [L, Hk, D]
            for h in range(hq):
                kh = h // (hq // hk)
                z = scale * (kk[:, kh] @ q[i, j, h])
                w = torch.softmax(z, 0)
                out[i, j, h] = w @ vv[:, kh]
                mag[i, j, h] = w @ vv[:, kh].abs()
                reach[i, j, h] = scale * (kk[:, kh].abs() @ q[i, j, h].abs()).max()
    return out, mag, reach


def decode_bound(out, mag, reach, d, dtype):
    """z = scale q.k: D fused multiply-adds and the scalings, (D + 8) U of the
    largest scale * sum |q k|, and the exponential's 2^-20; each enters the
    weights and their sum. The weights are held in two pieces of 8 bits or
    more: 2^-16. fp32 results: pieces of 11 bits, 2^-20."""
    z = 2 * ((d + 8) * U * reach + 2.0 ** -20 + (2.0 ** -20 if dtype == torch.float32 else 2.0 ** -16))
    return z.unsqueeze(-1) * mag + store_ulp(dtype) * out.abs() + tiny(dtype)


def assert_within(got, want, bound, what=""):
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(err).all(), f"{what}: not finite"
    over = err - bound
    assert (over <= 0).all(), f"{what}: {int((over > 0).sum())} of {over.numel()} outside; worst error " \
                              f"{err.flatten()[over.argmax()]:.3e} against {bound.expand_as(err).flatten()[over.argmax()]:.3e}"
