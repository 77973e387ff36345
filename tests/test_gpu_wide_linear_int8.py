"""GPU parity of the 8-bit linear layer. The sum of codes is exact, so a result
is off by the roundings of the int32 sum to fp32, of its products with the two
scales (the second fused with the bias) and of the activation and the store:

  |error| <= 3 U |acc sa sw| + U |y|  before the activation (U = 2^-24)

ReLU adds nothing, GELU passes an error on by at most 1.13 (its largest slope)
and is itself off by the error of erff (2 ulp: 2^-23 of at most 1, and the two
products): 2^-22 |y| for fp32 results. For 16-bit results it is max(x, 0) - a Q(a),
a = |x|, with Q off by 9e-6 of itself by its polynomial (test_block_host), by
46 * 2^-24 ln 2 = 2e-6 by the rounding of an exponent of up to 46, and by 2^-22 by
ex2.approx: 1.2e-5 a Q(a); past a = 8, a Q(a) < 5e-15 may be off by itself. The last
step rounds to 2^-24 |y| and the two terms."""
import math

import pytest
import torch

import block_ref as R
from gpu_util import no_device_error
from wide_compiler import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def case(n, rows, k, o, dtype, bias, seed=0):
    gen = torch.Generator().manual_seed(seed + k + o)
    codes = torch.randint(-127, 128, (n, *rows, k), generator=gen, dtype=torch.int8)
    w = torch.randint(-127, 128, (n, o, k), generator=gen, dtype=torch.int8)
    scale = torch.rand(n, *rows, generator=gen) * 0.02 + 1e-3
    ws = torch.rand(n, o, generator=gen) * 0.01 + 1e-4
    b = (torch.randn(n, o, generator=gen)).to(dtype) if bias else None
    return codes, scale, w, ws, b


def expect(codes, scale, w, ws, bias, act, dtype):
    n, k = w.shape[0], w.shape[2]
    acc = torch.matmul(codes.reshape(n, -1, k).double(), w.double().transpose(1, 2))
    prod = acc * scale.double().reshape(n, -1, 1) * ws.double()[:, None]
    y = prod if bias is None else prod + bias.double()[:, None]
    err = 3 * R.U * prod.abs() + R.U * y.abs()
    if act == ops.ACT_RELU:
        y = y.clamp(min=0)
    elif act == ops.ACT_GELU:
        own = 2.0 ** -22 * y.abs()
        if dtype != F32:
            tail = y.abs() * torch.special.erfc(y.abs() / math.sqrt(2)) / 2
            own = 1.2e-5 * tail + 5e-15 + 2 * R.U * y.abs()
        err = 1.13 * err + own
        y = torch.nn.functional.gelu(y)
    shape = (*codes.shape[:-1], w.shape[1])
    return y.view(shape), R.rounded(y, err, dtype).view(shape)


def held(t):
    """On the GPU with rows 16 bytes apart, what lies between them not zero."""
    k = t.shape[-1]
    wide = torch.full((*t.shape[:-1], -(-k // 16) * 16), 77, dtype=torch.int8, device=DEV)
    wide[..., :k] = t.to(DEV)
    return wide[..., :k]


def check(n, rows, k, o, dtype, bias=True, act=ops.ACT_NONE, keep=held):
    codes, scale, w, ws, b = case(n, rows, k, o, dtype, bias)
    y = ops.linear_int8(keep(codes), scale.to(DEV), keep(w), ws.to(DEV), None if b is None else b.to(DEV), act, dtype)
    want, bound = expect(codes, scale, w, ws, b, act, dtype)
    assert y.dtype == dtype and y.is_contiguous()
    R.assert_within(y, want, bound, f"{n} x {rows} x {k} -> {o}")
    no_device_error()


# few tokens: one to 128 (and past a tile of them), K in parts of one block and
# less, output channels that end inside a tile
@pytest.mark.parametrize("m", [1, 2, 7, 16, 17, 32, 40, 64, 65, 128, 131])
@pytest.mark.parametrize("k, o", [(1, 1), (16, 16), (33, 130), (128, 128), (129, 64), (512, 257), (1000, 96), (2048, 512)])
def test_few_tokens(m, k, o):
    check(2, (m,), k, o, BF16)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("act", [ops.ACT_NONE, ops.ACT_RELU, ops.ACT_GELU])
@pytest.mark.parametrize("bias", [False, True])
def test_types_and_activations(dtype, act, bias):
    check(3, (5,), 200, 150, dtype, bias, act)              # narrow
    check(40, (257,), 200, 264, dtype, bias, act)           # wide
    check(40, (300,), 72, 261, dtype, bias, act)            # wide, rows of y that 16-byte stores do not fit


# many rows: 256 x 256 tiles, their ends, several tiles a pair of SMs
@pytest.mark.parametrize("n, m, k, o", [(1, 4096, 256, 1024), (2, 1000, 333, 2000), (64, 129, 128, 256), (9, 640, 1024, 768),
                                        (37, 256, 64, 256), (1, 9000, 128, 520), (5, 513, 2064, 1032)])
def test_many_rows(n, m, k, o):
    for dtype in (BF16, F32):
        check(n, (m,), k, o, dtype)


def test_split_sums_reach_the_limits():
    """Longest K with codes at their ends: the sum stays within int32; the split
    over CTAs and their clusters gives it exactly."""
    k = 131071
    for m, code in ((1, 127), (3, -128)):
        codes = torch.full((1, m, k), code, dtype=torch.int8)
        w = torch.full((1, 5, k), -128, dtype=torch.int8)
        one = torch.ones(1, max(m, 5), device=DEV)
        y = ops.linear_int8(held(codes), one[:, :m].contiguous(), held(w), one[:, :5].contiguous(), dtype=F32)
        want = torch.tensor(float(code * -128 * k), dtype=torch.float64)
        assert ((y.double().cpu() - want).abs() <= want.abs() * R.U).all()


def test_leading_dims_and_strides():
    codes, scale, w, ws, b = case(2, (3, 4, 5), 48, 96, BF16, True)
    want, bound = expect(codes, scale, w, ws, b, ops.ACT_NONE, BF16)
    args = (scale.to(DEV), w.to(DEV), ws.to(DEV), b.to(DEV))
    c = codes.to(DEV)
    views = [c, c.transpose(1, 2).contiguous().transpose(1, 2),
             torch.cat([c, c], -1)[..., 48:], torch.cat([c, c], 1)[:, 3:], c.flip(0).flip(0)]
    odd = torch.zeros(c.numel() + 1, dtype=torch.int8, device=DEV)
    odd[1:] = c.flatten()
    views.append(odd[1:].view(c.shape))
    for v in views:
        R.assert_within(ops.linear_int8(v, *args), want, bound)
    wt = w.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    R.assert_within(ops.linear_int8(c, args[0], wt, args[2], args[3]), want, bound)
    st = args[0].transpose(0, 1).contiguous().transpose(0, 1)
    R.assert_within(ops.linear_int8(c, st, args[1], args[2], args[3]), want, bound)


def test_one_model_for_all_rows_expanded():
    """A weight that the models share (an expanded view)."""
    codes, scale, w, ws, _ = case(1, (6,), 64, 80, F32, False)
    c3, s3 = codes.expand(3, -1, -1).contiguous(), scale.expand(3, -1).contiguous()
    y = ops.linear_int8(held(c3), s3.to(DEV), held(w).expand(3, -1, -1), ws.expand(3, -1).to(DEV), dtype=F32)
    want, bound = expect(codes, scale, w, ws, None, ops.ACT_NONE, F32)
    R.assert_within(y, want.expand(3, -1, -1), bound.expand(3, -1, -1))


def test_rows_that_are_not_finite_stay_apart():
    codes, scale, w, ws, _ = case(1, (4,), 64, 80, BF16, False)
    scale[0, 1], scale[0, 2] = math.inf, math.nan
    codes[0, 1:3] = 0                                   # as quantize_rows makes them
    for act in (ops.ACT_NONE, ops.ACT_RELU, ops.ACT_GELU):
        for dtype in (BF16, F32):
            y = ops.linear_int8(held(codes), scale.to(DEV), held(w), ws.to(DEV), act=act, dtype=dtype)
            assert y[0, 1].isnan().all() and y[0, 2].isnan().all() and y[0, [0, 3]].isfinite().all()


def test_nothing_to_compute():
    z = lambda *s: torch.zeros(*s, dtype=torch.int8, device=DEV)
    f = lambda *s: torch.zeros(*s, device=DEV)
    assert ops.linear_int8(z(2, 0, 16), f(2, 0), z(2, 5, 16), f(2, 5)).shape == (2, 0, 5)
    assert ops.linear_int8(z(0, 3, 16), f(0, 3), z(0, 5, 16), f(0, 5)).shape == (0, 3, 5)
    assert ops.linear_int8(z(2, 3, 16), f(2, 3), z(2, 0, 16), f(2, 0)).shape == (2, 3, 0)
    with pytest.raises(ValueError, match="k from 1"):
        ops.linear_int8(z(2, 3, 0), f(2, 3), z(2, 5, 0), f(2, 5))


def test_two_streams_and_a_graph():
    args = []
    for seed in range(2):
        codes, scale, w, ws, b = case(4, (3,), 1024, 512, BF16, True, seed)
        args.append((held(codes), scale.to(DEV), held(w), ws.to(DEV), b.to(DEV)))
    want = [ops.linear_int8(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(20):
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                outs.append(ops.linear_int8(*a))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(outs))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.linear_int8(*args[0])
    args[0][0].copy_(args[1][0])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, ops.linear_int8(*args[0]))
    no_device_error()


@pytest.mark.parametrize("rows", [(3, 1), (2, 200)])
def test_a_served_feed_forward(rows):
    """Norm, codes, up + GELU, codes, down, as a layer runs them: against the
    same steps in 64 bits on the codes that each step really made."""
    n, d, hidden = 2, 264, 520
    gen = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen).to(BF16).to(DEV)
    x, y, pw = rand(n, *rows, d), rand(n, *rows, d), 1 + 0.2 * rand(n, d)
    up, us = ops.quantize_rows(rand(n, hidden, d) / math.sqrt(d))
    down, ds = ops.quantize_rows(rand(n, d, hidden) / math.sqrt(hidden))
    h, codes, scale = ops.residual_norm_quantize(x, y, pw, post_weight=pw)
    a = ops.linear_int8(codes, scale, up, us, act=ops.ACT_GELU)
    c2, s2 = ops.quantize_rows(a)
    out = ops.linear_int8(c2, s2, down, ds)
    ref = R.residual_norm(x.cpu(), y.cpu(), pw.cpu(), post_weight=pw.cpu())
    R.assert_within(h, *ref["h"])
    s, es, q, eq = R.codes(*ref["z32"])
    R.assert_within(codes, q, 0.5 + eq)
    R.assert_within(a, *expect(codes.cpu(), scale.cpu(), up.cpu(), us.cpu(), None, ops.ACT_GELU, BF16))
    R.assert_within(c2, a.cpu().double() / s2.cpu().double()[..., None], torch.full(c2.shape, 0.5 + 128 * R.U))
    R.assert_within(out, *expect(c2.cpu(), s2.cpu(), down.cpu(), ds.cpu(), None, ops.ACT_NONE, BF16))


def test_offsets_past_32_bits():
    """Rows of results past 2^31 values, and codes past 2^31."""
    m, k, o = 270000, 64, 8192
    codes, scale, w, ws, _ = case(1, (1,), k, o, BF16, False)
    many = codes.to(DEV).expand(1, m, k).contiguous()
    s = scale.to(DEV).expand(1, m).contiguous()
    s[0, -1] *= 2
    y = ops.linear_int8(many, s, w.to(DEV), ws.to(DEV))
    want, bound = expect(codes, scale, w, ws, None, ops.ACT_NONE, BF16)
    for row, f in ((0, 1), (m // 2, 1), (m - 2, 1), (m - 1, 2)):
        R.assert_within(y[:, row:row + 1], want * f, bound * f)
    del y
    k = 131056
    big = torch.ones(1, 17000, k, dtype=torch.int8, device=DEV)
    big[0, -1] = -3
    one = torch.ones(1, 17000, device=DEV)
    wide = torch.ones(1, 20, k, dtype=torch.int8, device=DEV)
    for y in (ops.linear_int8(big, one, wide, one[:, :20].contiguous(), dtype=F32),
              ops.linear_int8(wide, one[:, :20].contiguous(), big, one, dtype=F32).transpose(1, 2)):
        assert (y[0, :-1] == k).all() and (y[0, -1] == -3 * k).all()
    no_device_error()
