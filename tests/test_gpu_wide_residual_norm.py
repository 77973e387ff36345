"""GPU parity of the residual norm (forward, 8-bit codes, gradients) and of the
row quantiser against the 64-bit formulas of block_ref, with its bounds."""
import math

import pytest
import torch

import block_ref as R
from gpu_util import no_device_error
from wide_compiler import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = ("x", "y", "weight", "bias", "post_weight", "post_bias", "gate")


def tensors(shape, dtype, center, post, gate, seed, y=True, device=DEV):
    """The seven tensors by name (None where there is none)."""
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)
    n, d = shape[0], shape[-1]
    out = dict.fromkeys(NAMES)
    out["x"] = rand(*shape) * 2 + 0.5
    out["weight"] = 1 + 0.3 * rand(n, d)
    out["bias"] = 0.2 * rand(n, d) if center else None
    if y:
        out["y"] = rand(*shape) * torch.exp(rand(n, *(1,) * (len(shape) - 2), d))
        if post:
            out["post_weight"] = 1 + 0.3 * rand(n, d)
            out["post_bias"] = 0.2 * rand(n, d) if center else None
        if gate is not None:
            out["gate"] = 0.7 + 0.4 * rand(*shape[:1 + gate], d)
    return {k: None if v is None else v.to(dtype).to(device) for k, v in out.items()}


def cpu(t):
    return {k: None if v is None else v.detach().cpu() for k, v in t.items()}


# [N, ..., D]: sizes where the vector, the threads of a row and the values a
# thread holds change, odd ones among them
SHAPES = [(1, 1, 1), (2, 3, 7), (3, 2, 5, 64), (1, 4, 256), (2, 5, 260), (2, 2, 3, 500), (2, 3, 501), (1, 9, 1024),
          (2, 3, 1032), (2, 2, 2, 2050), (1, 3, 4096), (1, 2, 4100), (2, 2, 4101), (1, 3, 8192), (2, 8)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("center", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, center, dtype):
    for k, (post, gate) in enumerate([(True, 0), (False, None), (True, None), (False, len(shape) - 2)]):
        t = tensors(shape, dtype, center, post, gate, sum(shape) + k)
        want = R.residual_norm(**cpu(t), scale=0.75, center=center)
        h, z = ops.residual_norm(**t, scale=0.75, center=center)
        assert h.dtype == z.dtype == dtype and h.shape == z.shape == shape
        R.assert_within(h, *want["h"], "h")
        R.assert_within(z, *want["z"], "z")
    no_device_error()


@pytest.mark.parametrize("rows", [1, 3, 5000])
@pytest.mark.parametrize("d", [192, 1000, 2048])
def test_forward_few_and_many_rows(rows, d):
    """Few rows are spread over more threads than many."""
    t = tensors((2, rows, d), BF16, False, True, 0, rows + d)
    want = R.residual_norm(**cpu(t))
    h, z = ops.residual_norm(**t)
    R.assert_within(h, *want["h"], "h")
    R.assert_within(z, *want["z"], "z")


# rows enough for 16 channels (norms) and 32 (codes) a thread, in every vector and team
MANY = [(1, 60000, 60), (2, 15000, 104), (1, 20000, 250), (3, 4000, 501), (1, 9000, 1000), (2, 800, 4092), (1, 700, 8190)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("center", [False, True])
@pytest.mark.parametrize("shape", MANY)
def test_many_rows_of_every_kind(shape, center, dtype):
    t = tensors(shape, dtype, center, True, 1 if shape[2] < 300 else 0, sum(shape))
    want = R.residual_norm(**cpu(t), center=center)
    h, z = ops.residual_norm(**t, center=center)
    R.assert_within(h, *want["h"], "h")
    R.assert_within(z, *want["z"], "z")
    h, codes, scales = ops.residual_norm_quantize(**t, center=center)
    R.assert_within(h, *want["h"], "h")
    check_codes(*want["z32"], codes, scales, shape[-1])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", MANY + [(1, 300, 16384), (1, 400, 16380), (2, 300, 16383)])
def test_codes_of_many_rows(shape, dtype):
    x = torch.randn(*shape, device=DEV).to(dtype)
    x[0, 5, shape[-1] // 2] = -50
    codes, scales = ops.quantize_rows(x)
    top = x.float().abs().amax(-1).clamp(min=2.0 ** -40)
    want = top / torch.full_like(top, 127.0)
    assert torch.equal(scales, want)
    assert torch.equal(codes.float(), torch.round(x.float() / want.unsqueeze(-1)))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("center", [False, True])
def test_without_y_h_is_x(center, dtype):
    t = tensors((2, 3, 100), dtype, center, False, None, 5, y=False)
    h, z = ops.residual_norm(**t, center=center)
    assert h is t["x"]
    R.assert_within(z, *R.residual_norm(**cpu(t), center=center)["z"], "z")


def test_other_strides_and_offsets():
    """Transposed and offset inputs give what dense copies give."""
    t = tensors((2, 3, 4, 96), BF16, False, True, 2, 9)
    want = ops.residual_norm(**t)
    wide = torch.randn(2, 3, 4, 100, device=DEV).to(BF16)
    wide[..., 3:99] = t["y"]
    moved = dict(t, x=t["x"].transpose(1, 2).contiguous().transpose(1, 2), y=wide[..., 3:99])
    for a, b in zip(ops.residual_norm(**moved), want):
        assert torch.equal(a, b)
    flat = torch.empty(2 * 3 * 4 * 96 + 1, device=DEV, dtype=BF16)
    flat[1:] = t["x"].flatten()
    h, z = ops.residual_norm(**dict(t, x=flat[1:].view(2, 3, 4, 96)))      # 2-byte aligned: one value at a time
    ref = R.residual_norm(**cpu(t))
    R.assert_within(h, *ref["h"], "h")
    R.assert_within(z, *ref["z"], "z")


def test_rows_of_zeros_and_equal_values():
    t = tensors((2, 4, 72), F32, True, True, None, 3)
    t["x"][0, 1], t["y"][0, 1] = 0, 0
    t["x"][1, 2], t["y"][1, 2] = 5, 0
    for center in (False, True):
        if not center:
            t["bias"] = t["post_bias"] = None
        want = R.residual_norm(**cpu(t), center=center)
        h, z = ops.residual_norm(**t, center=center)
        assert torch.isfinite(z).all()
        R.assert_within(h, *want["h"], "h")
        R.assert_within(z, *want["z"], "z")
        t["bias"] = t["post_bias"] = torch.zeros(2, 72, device=DEV)


def test_no_rows():
    t = tensors((2, 0, 64), BF16, False, True, 1, 1)
    h, z = ops.residual_norm(**t)
    assert h.shape == z.shape == (2, 0, 64)
    h, codes, scales = ops.residual_norm_quantize(**t)
    assert codes.shape == (2, 0, 64) and scales.shape == (2, 0)
    codes, scales = ops.quantize_rows(t["x"])
    assert codes.shape == (2, 0, 64)
    codes, scales = ops.quantize_rows(torch.empty(3, 0, device=DEV))
    assert codes.shape == (3, 0) and torch.equal(scales, torch.full((3,), 2.0 ** -40 / 127, device=DEV))


def check_codes(z, ez, codes, scales, k):
    s, es, q, eq = R.codes(z, ez)
    R.assert_within(scales, s, es, "scales")
    R.assert_within(codes, q, 0.5 + eq, "codes")
    assert codes.dtype == torch.int8 and codes.stride(-2) % 16 == 0 and codes.shape[-1] == k


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("center", [False, True])
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 7), (3, 2, 5, 64), (2, 5, 260), (2, 3, 501), (2, 700, 1024),
                                   (1, 3, 4100), (1, 2, 8192)])
def test_codes_of_the_norm(shape, center, dtype):
    t = tensors(shape, dtype, center, True, 0, sum(shape))
    want = R.residual_norm(**cpu(t), center=center)
    h, codes, scales = ops.residual_norm_quantize(**t, center=center)
    R.assert_within(h, *want["h"], "h")
    check_codes(*want["z32"], codes, scales, shape[-1])
    t = tensors(shape, dtype, center, False, None, 1, y=False)
    h, codes, scales = ops.residual_norm_quantize(**t, center=center)
    assert h is t["x"]
    check_codes(*R.residual_norm(**cpu(t), center=center)["z32"], codes, scales, shape[-1])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1,), (3, 1), (5, 16), (2, 3, 333), (4, 1000), (3, 1, 1024), (300, 2048), (2, 5, 4098),
                                   (3, 32768), (2, 40007), (1, 65536)])
def test_quantize_rows(shape, dtype):
    """Largest value exact, scale and quotient rounded once each: equal codes."""
    gen = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(*shape, generator=gen) * torch.exp(2 * torch.randn(*shape[:-1], 1, generator=gen))).to(dtype)
    if len(shape) > 1:
        x[0] = 0
    codes, scales = ops.quantize_rows(x.to(DEV))
    top = x.float().abs().amax(-1).clamp(min=2.0 ** -40)
    want = top / torch.full_like(top, 127.0)
    assert torch.equal(scales.cpu(), want)
    assert torch.equal(codes.cpu().float(), torch.round(x.float() / want.unsqueeze(-1)))
    assert len(shape) < 2 or codes.stride(-2) % 16 == 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(20001, 130), (10007, 258), (9001, 333), (5003, 500), (2503, 1000), (1201, 2050),
                                   (701, 4096), (401, 8192), (301, 8200), (201, 9001), (205, 12290), (151, 16384)])
def test_quantize_many_rows(shape, dtype):
    """Every count of values a thread, with several rows a team: the quotients of the
    largest value and of the values, rounded once each."""
    gen = torch.Generator(device=DEV).manual_seed(sum(shape))
    x = torch.randn(*shape, generator=gen, device=DEV)
    x = (x * torch.exp(2 * torch.randn(shape[0], 1, generator=gen, device=DEV))).to(dtype)
    codes, scales = ops.quantize_rows(x)
    x = x.cpu().float()
    top = x.abs().amax(-1).clamp(min=2.0 ** -40)
    want = top / torch.full_like(top, 127.0)
    assert torch.equal(scales.cpu(), want)
    assert torch.equal(codes.cpu().float(), torch.round(x / want.unsqueeze(-1)))


def test_rows_that_are_not_finite():
    x = torch.randn(4, 50, device=DEV)
    x[1, 7], x[2, 3] = math.inf, math.nan
    codes, scales = ops.quantize_rows(x)
    assert scales[1] == math.inf and scales[2].isnan() and scales[[0, 3]].isfinite().all()
    assert not codes[1].any() and not codes[2].any()
    w = torch.ones(1, 50, device=DEV)
    _, codes, scales = ops.residual_norm_quantize(x[None], None, w)
    assert not scales[0, 1].isfinite() and scales[0, 2].isnan() and scales[0, [0, 3]].isfinite().all()


# ---------------------------------------------------------------------------
# Gradients
# ---------------------------------------------------------------------------

GRAD_NAMES = dict(x="dx", y="dy", weight="dweight", bias="dbias", post_weight="dpost_weight", post_bias="dpost_bias",
                  gate="dgate")


def check_grads(t, dh, dz, scale, center):
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items() if v is not None}
    h, z = ops.residual_norm(**{**t, **leaves}, scale=scale, center=center)
    outs, gs = zip(*[(o, g) for o, g in ((h, dh), (z, dz)) if g is not None])
    grads = torch.autograd.grad(outs, list(leaves.values()), gs, allow_unused=True)
    want = R.residual_norm(**cpu(t), scale=scale, center=center, dh=None if dh is None else dh.cpu(),
                           dz=None if dz is None else dz.cpu())
    R.assert_within(h, *want["h"], "h")
    R.assert_within(z, *want["z"], "z")
    for (name, leaf), g in zip(leaves.items(), grads):
        assert g.shape == leaf.shape and g.dtype == leaf.dtype
        R.assert_within(g, *want[GRAD_NAMES[name]], GRAD_NAMES[name])


@pytest.mark.grad
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("center", [False, True])
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 7), (3, 2, 5, 64), (1, 4, 256), (2, 5, 260), (2, 2, 3, 500),
                                   (2, 3, 501), (1, 40, 1024), (2, 2, 2, 2050), (1, 3, 4096), (2, 2, 4101), (2, 3, 4104),
                                   (1, 2, 8192), (2, 8)])
def test_gradients(shape, center, dtype):
    gen = torch.Generator().manual_seed(sum(shape))
    dh, dz = (torch.randn(*shape, generator=gen).to(dtype).to(DEV) for _ in range(2))
    for k, (post, gate) in enumerate([(True, 0), (False, None), (True, len(shape) - 2), (False, 0), (True, None)]):
        t = tensors(shape, dtype, center, post, gate, sum(shape) + k)
        check_grads(t, dh, dz, 0.75, center)
    no_device_error()


# a gate for each sequence: walks that hold many sequences, one, or a part of one
@pytest.mark.grad
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("center", [False, True])
@pytest.mark.parametrize("shape", [(1, 2, 3, 64), (2, 3, 1000, 32), (1, 700, 3, 40), (3, 5, 77, 501), (2, 4000, 2, 8),
                                   (1, 1, 50, 72), (2, 3, 40, 4200), (16, 9, 40, 320)])
def test_gradients_with_a_gate_for_each_sequence(shape, center, dtype):
    gen = torch.Generator().manual_seed(sum(shape))
    dh, dz = (torch.randn(*shape, generator=gen).to(dtype).to(DEV) for _ in range(2))
    for post in (True, False):
        check_grads(tensors(shape, dtype, center, post, 1, sum(shape)), dh, dz, 1.0, center)


@pytest.mark.grad
@pytest.mark.parametrize("center", [False, True])
def test_gradients_of_one_output_and_without_y(center):
    shape = (2, 3, 5, 120)
    dz = torch.randn(*shape, device=DEV)
    for gate in (None, 0, 1, 2):
        t = tensors(shape, F32, center, True, gate, 11)
        check_grads(t, None, dz, 0.5, center)
        check_grads(t, dz, None, 0.5, center)
    t = tensors(shape, F32, center, False, None, 12, y=False)
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items() if v is not None}
    h, z = ops.residual_norm(**{**t, **leaves}, center=center)
    assert h is leaves["x"]
    grads = torch.autograd.grad((h, z), list(leaves.values()), (dz, dz))
    want = R.residual_norm(**cpu(t), center=center, dz=dz.cpu())
    R.assert_within(grads[0] - dz, want["dx"][0], want["dx"][1] + 4 * R.U * dz.cpu().abs().double(), "dx")
    R.assert_within(grads[1], *want["dweight"], "dweight")


@pytest.mark.grad
def test_gradients_of_many_rows_are_the_same_each_time():
    t = tensors((4, 3, 900, 256), BF16, True, True, 1, 2)
    leaves = {k: v.requires_grad_(True) for k, v in t.items() if v is not None}
    g = torch.randn_like(t["x"])
    h, z = ops.residual_norm(**t, center=True)
    a = torch.autograd.grad((h, z), list(leaves.values()), (g, g), retain_graph=True)
    b = torch.autograd.grad((h, z), list(leaves.values()), (g, g))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.grad
def test_some_gradients_only():
    """Frozen parameters, and parameters alone."""
    t = tensors((2, 3, 4, 96), F32, False, True, 0, 8)
    g = torch.randn_like(t["x"])
    full = {k: v.clone().requires_grad_(True) for k, v in t.items() if v is not None}
    want = dict(zip(full, torch.autograd.grad(ops.residual_norm(**{**t, **full}), list(full.values()), (g, g))))
    for some in (("x",), ("y",), ("weight",), ("gate",), ("post_weight", "y"), ("x", "weight")):
        leaves = {k: t[k].clone().requires_grad_(True) for k in some}
        h, z = ops.residual_norm(**{**t, **leaves})
        got = torch.autograd.grad((h, z), list(leaves.values()), (g, g))
        assert all(torch.equal(a, want[k]) for a, k in zip(got, some))


@pytest.mark.grad
def test_differences():
    """Directional derivatives of a fp32 sum against central differences of the
    64-bit formula (their own error: step^2, far below 1e-3)."""
    t = tensors((2, 3, 5, 60), F32, True, True, 1, 21)
    gen = torch.Generator().manual_seed(4)
    dh, dz = (torch.randn(2, 3, 5, 60, generator=gen) for _ in range(2))
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    h, z = ops.residual_norm(**leaves, scale=0.6, center=True)
    grads = torch.autograd.grad((h, z), list(leaves.values()), (dh.to(DEV), dz.to(DEV)))
    base = {k: v.double() for k, v in cpu(t).items()}

    def value(p):
        out = R.residual_norm(**p, scale=0.6, center=True)
        return float((out["h"][0] * dh.double()).sum() + (out["z"][0] * dz.double()).sum())

    for k, g in zip(leaves, grads):
        step = torch.randn(base[k].shape, generator=gen, dtype=torch.float64) * 1e-4
        slope = (value({**base, k: base[k] + step}) - value({**base, k: base[k] - step})) / 2
        assert math.isclose(float((g.cpu().double() * step).sum()), slope, rel_tol=1e-3, abs_tol=1e-6), k


@pytest.mark.grad
def test_gradients_of_gradients():
    t = tensors((2, 2, 3, 24), F32, True, True, 1, 30)
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    outs = ops.residual_norm(**leaves, center=True)
    gx = torch.autograd.grad(outs[1].sum() + (outs[0] ** 2).sum(), leaves["x"], create_graph=True)[0]
    got = torch.autograd.grad((gx ** 2).sum(), list(leaves.values()))
    d = {k: v.detach().double().requires_grad_(True) for k, v in leaves.items()}
    norm = lambda v, w, b: (torch.nn.functional.layer_norm(v, (24,), eps=1e-6) * w[:, None, None] + b[:, None, None])
    h = d["x"] + d["gate"][:, :, None] * norm(d["y"], d["post_weight"], d["post_bias"])
    gx = torch.autograd.grad(norm(h, d["weight"], d["bias"]).sum() + (h ** 2).sum(), d["x"], create_graph=True)[0]
    want = torch.autograd.grad((gx ** 2).sum(), list(d.values()), allow_unused=True)
    for a, b in zip(got, want):
        b = torch.zeros_like(a) if b is None else b
        torch.testing.assert_close(a.double(), b.double(), rtol=1e-3, atol=1e-3)


# ---------------------------------------------------------------------------
# Streams and graphs
# ---------------------------------------------------------------------------

@pytest.mark.grad
def test_captured_step_replays():
    """Forward and backward captured into a graph and replayed on new values."""
    t = tensors((2, 3, 50, 264), BF16, False, True, 1, 40)
    leaves = [v.requires_grad_(True) for v in t.values() if v is not None]
    g = torch.randn_like(t["x"])

    def step():
        h, z = ops.residual_norm(**t)
        return h, z, *torch.autograd.grad((h, z), leaves, (g, g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        t["x"].normal_()
        t["y"].normal_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


def test_another_stream():
    t = tensors((2, 64, 2048), BF16, False, True, 0, 41)
    want = ops.residual_norm(**t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.residual_norm(**t)
        codes, scales = ops.quantize_rows(got[1])
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(codes, ops.quantize_rows(want[1])[0])


# ---------------------------------------------------------------------------
# Far offsets, threads, call history
# ---------------------------------------------------------------------------

def test_offsets_past_32_bits():
    """The last rows of tensors of over 2^31 values are what a call on them alone
    gives."""
    n, rows, d = 1, 270000, 8192
    t = {k: torch.randn(n, rows, d, device=DEV, dtype=BF16) for k in ("x", "y")}
    w = 1 + 0.2 * torch.randn(n, d, device=DEV, dtype=BF16)
    h, z = ops.residual_norm(t["x"], t["y"], w, post_weight=w)
    last = {k: v[:, -5:].contiguous() for k, v in t.items()}
    h2, z2 = ops.residual_norm(last["x"], last["y"], w, post_weight=w)
    ref = R.residual_norm(last["x"].cpu(), last["y"].cpu(), w.cpu(), post_weight=w.cpu())
    for got, alone, name in ((h[:, -5:], h2, "h"), (z[:, -5:], z2, "z")):
        R.assert_within(got, *ref[name], name)
        R.assert_within(alone, *ref[name], name)
    del h
    codes, scales = ops.quantize_rows(z)
    c2, s2 = ops.quantize_rows(z[:, -5:].contiguous())
    assert torch.equal(codes[:, -5:], c2) and torch.equal(scales[:, -5:], s2)
    _, codes, scales = ops.residual_norm_quantize(t["x"], t["y"], w, post_weight=w)
    s, es, q, eq = R.codes(*ref["z32"])
    R.assert_within(scales[:, -5:], s, es, "scales")
    R.assert_within(codes[:, -5:], q, 0.5 + eq, "codes")


@pytest.mark.grad
def test_gradients_do_not_depend_on_earlier_calls():
    """The split of the sums is the sizes' alone: rows of 240 (lanes of a warp) and of
    1000 channels (a block of as many threads) in both orders."""
    def grads(d):
        t = tensors((3, 4, 500, d), BF16, False, True, 0, d)
        leaves = [v.requires_grad_(True) for v in t.values() if v is not None]
        out = ops.residual_norm(**t)
        return torch.autograd.grad(out, leaves, (t["x"].detach(), t["y"].detach()))

    a = grads(240), grads(1000)
    b = grads(1000), grads(240)
    assert all(torch.equal(x, y) for x, y in zip((*a[0], *a[1]), (*b[1], *b[0])))


def test_calls_from_several_threads():
    import threading
    sizes = [(2, 300, 1024), (2, 40, 8192), (2, 300, 200), (2, 90, 3000)]
    args = [tensors(s, F32, True, True, 0, i) for i, s in enumerate(sizes)]
    want = [ops.residual_norm(**t, center=True) for t in args]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        s = torch.cuda.Stream()
        try:
            with torch.cuda.stream(s):
                for _ in range(50):
                    got = ops.residual_norm(**args[i], center=True)
                    codes, _ = ops.quantize_rows(got[1])
            s.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                failed.append(i)
        except Exception as e:           # reported by the main thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sizes))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed
