"""What is measured of the operators around a decoder block of N fused models:
the norms of the residual stream, and linear layers in 8-bit integers.

Five paths, each as its plain form (elementary torch operations in 32 bits)
and as the calls a user makes of ``wide_compiler``:

  norm     the residual stream after a block, and the norm before the next:
             u = norm(y) or y,  h = x + scale * gate * u,  z = norm(h)
  train    the same with all its gradients
  linear8  a linear layer on 8-bit codes: one scale a token, one an output channel
  proj8    the norm of the residual stream straight into codes, and a linear layer on them
  mlp8     a served feed-forward block: norm, codes, up, GELU, codes, down

Tensors are N-first: x, y, h, z [N, B, T, D], norm weights [N, D], gates [N, D]
(one for each model), [N, B, D] (each sequence) or [N, B, T, D] (each token),
linear weights [N, O, K] as int8 codes with float32 scales [N, O].
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
FLOOR = 2.0 ** -40          # smallest row maximum that codes are scaled by


def listed():
    return [
        # a training step of the block boundary: RMS norms on both sides, a learned gate for each model
        dict(name="train_bf16", kind="train", dtype="bf16", n=8, b=4, t=1024, d=1024, center=False, post=True,
             gate="model", scale=1.0),
        # odd sizes, LayerNorm with biases, a gate for each sequence, 32-bit gradients
        dict(name="train_f32_odd", kind="train", dtype="f32", n=3, b=5, t=77, d=501, center=True, post=True,
             gate="sequence", scale=0.7),
        # few wide models, LayerNorm before each block only
        dict(name="train_f16_wide", kind="train", dtype="f16", n=2, b=2, t=1024, d=4096, center=True, post=False,
             gate="none", scale=1.0),
        # one token of every sequence: latency
        dict(name="norm_token_bf16", kind="norm", dtype="bf16", n=8, b=4, t=1, d=1024, center=False, post=True,
             gate="none", scale=0.5),
        # prompts of several models: throughput
        dict(name="norm_prompt_bf16", kind="norm", dtype="bf16", n=8, b=4, t=2048, d=2048, center=False, post=True,
             gate="model", scale=1.0),
        # one token: norm into codes, then the fused projection of 16 query and 4 key heads of 64
        dict(name="proj8_token_bf16", kind="proj8", dtype="bf16", n=8, b=4, t=1, d=1024, o=1536, center=False,
             post=False, gate="none", scale=1.0, bias=False),
        # prompts: norms of both sides into codes, then a fused projection
        dict(name="proj8_prompt_f16", kind="proj8", dtype="f16", n=4, b=4, t=512, d=2048, o=2560, center=False,
             post=True, gate="model", scale=1.0, bias=True),
        # one token of a small batch through a wide layer: the weights are read once
        dict(name="linear8_token_bf16", kind="linear8", dtype="bf16", n=8, b=4, t=1, k=1024, o=4096, act="gelu",
             bias=True),
        # the benchmark's linear layer (64 models, batch 256, 1024 -> 1024) in 8 bits
        dict(name="linear8_batch_bf16", kind="linear8", dtype="bf16", n=64, b=256, t=1, k=1024, o=1024, act="none",
             bias=True),
        # odd sizes in 32 bits: rows of 333 codes, 517 output channels
        dict(name="linear8_f32_odd", kind="linear8", dtype="f32", n=3, b=37, t=1, k=333, o=517, act="relu", bias=True),
        # one decoder step of a batch through the feed-forward block
        dict(name="mlp8_step_bf16", kind="mlp8", dtype="bf16", n=8, b=32, t=1, d=1024, o=4096, center=False,
             post=True, gate="none", scale=1.0, bias=False),
        # prompts through the feed-forward block: the largest products
        dict(name="mlp8_prompt_bf16", kind="mlp8", dtype="bf16", n=8, b=4, t=1024, d=1024, o=4096, center=True,
             post=False, gate="none", scale=1.0, bias=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row's length: often a power of two, often a multiple of 8, else any."""
    r = rng.random()
    if r < 0.3:
        return rng.choice([1 << i for i in range(20) if lo <= 1 << i <= hi])
    w = _log(rng, lo, hi)
    return max(8, w // 8 * 8) if r < 0.7 else w


def draw(rng):
    kind = rng.choice(("train", "train", "norm", "linear8", "linear8", "proj8", "mlp8"))
    c = dict(kind=kind, n=_log(rng, 1, 64), b=_log(rng, 1, 64), t=rng.choice((1, _log(rng, 1, 2048))))
    # codes of a normalised row are compared as a 16-bit result: a tie of their rounding is a whole code
    c["dtype"] = rng.choice(("bf16", "f16", "f32") if kind in ("train", "norm", "linear8") else ("bf16", "f16"))
    if kind == "linear8":
        c.update(k=_width(rng, 16, 8192), o=_width(rng, 16, 8192), act=rng.choice(("none", "relu", "gelu")),
                 bias=rng.random() < 0.5)
    else:
        c.update(d=_width(rng, 16, 8192), center=rng.random() < 0.4, post=rng.random() < 0.5,
                 gate=rng.choice(("none", "model", "sequence", "token")), scale=rng.choice((1.0, 0.5, 0.22)))
        if kind in ("proj8", "mlp8"):
            c.update(o=_width(rng, 16, 8192), bias=rng.random() < 0.5)
    shrink = [k for k in ("t", "b", "n", "d", "k", "o") if k in c]
    while work(c)["bytes"] > 5e8 or work(c)["flops"] > 4e11 or _weights(c) > 2e8:
        k = max(shrink, key=lambda s: c[s])
        c[k] = max(1, c[k] * 2 // 3)
    return c


def _weights(c):
    """Codes of all linear weights (the plain form widens them)."""
    k = c.get("k", c.get("d", 0))
    return c["n"] * k * c["o"] * (2 if c["kind"] == "mlp8" else 1) if "o" in c else 0


# ---------------------------------------------------------------------------
# What a user's program has before the call
# ---------------------------------------------------------------------------

def _gate_shape(c):
    return {"model": (c["n"], c["d"]), "sequence": (c["n"], c["b"], c["d"]),
            "token": (c["n"], c["b"], c["t"], c["d"])}[c["gate"]]


def _codes(w):
    """A weight [N, O, K] as the program keeps it: int8 rows (16 bytes apart,
    or a multiple of that) and one scale for each output channel."""
    scale = w.abs().amax(-1).clamp(min=FLOOR) / torch.full(w.shape[:2], 127.0, device=DEV)
    k = w.shape[-1]
    held = torch.zeros(*w.shape[:2], -(-k // 16) * 16, device=DEV, dtype=torch.int8)
    held[..., :k] = torch.round(w / scale.unsqueeze(-1)).to(torch.int8)
    return held[..., :k], scale


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[c["dtype"]]
    rand = lambda *shape: torch.randn(*shape, device=DEV, generator=g)  # noqa: E731
    s = dict(c=c)

    def layer(o, k, bias):
        w, scale = _codes(rand(c["n"], o, k) / math.sqrt(k))
        return w, scale, (0.1 * rand(c["n"], o)).to(dt) if bias else None

    rows = (c["n"], c["b"], c["t"])
    if c["kind"] == "linear8":
        # activations have a few channels that are much larger than the rest
        s["x"] = (rand(*rows, c["k"]) * torch.exp(0.7 * rand(c["n"], 1, 1, c["k"]))).to(dt)
        s["layer"] = layer(c["o"], c["k"], c["bias"])
        return s
    d = c["d"]
    s["x"] = (2 * rand(*rows, d) * torch.exp(0.5 * rand(c["n"], 1, 1, d)) + 0.3).to(dt)
    s["y"] = (rand(*rows, d) * torch.exp(0.5 * rand(c["n"], 1, 1, d)) + 0.1).to(dt)
    norm = lambda: (1 + 0.2 * rand(c["n"], d)).to(dt)  # noqa: E731
    shift = lambda: (0.1 * rand(c["n"], d)).to(dt) if c["center"] else None  # noqa: E731
    s["weight"], s["weight_bias"] = norm(), shift()
    s["post"], s["post_bias"] = (norm(), shift()) if c["post"] else (None, None)
    s["gate"] = None if c["gate"] == "none" else (0.6 + 0.3 * rand(*_gate_shape(c))).to(dt)
    if c["kind"] == "train":
        s["dh"], s["dz"] = rand(*rows, d).to(dt), rand(*rows, d).to(dt)
        for k in _INPUTS:
            if s[k] is not None:
                s[k].requires_grad_(True)
    if c["kind"] == "proj8":
        s["layer"] = layer(c["o"], d, c["bias"])
    if c["kind"] == "mlp8":
        s["up"], s["down"] = layer(c["o"], d, c["bias"]), layer(d, c["o"], c["bias"])
    return s


_INPUTS = ("x", "y", "weight", "weight_bias", "post", "post_bias", "gate")


# ---------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------

def _over(w):
    """[N, D], [N, B, D] or [N, B, T, D] over the rows, in 32 bits."""
    return None if w is None else w.float().view(w.shape[:-1] + (1,) * (4 - w.dim()) + w.shape[-1:])


def _normed(v, center):
    """Normalised rows and the factor that made them so."""
    v = v - v.mean(-1, keepdim=True) if center else v
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    return v * r, r


def _affine(v, w, b):
    return v * w if b is None else v * w + b


def _plain_norm(s):
    """h, z and what their gradients need."""
    c = s["c"]
    y, x = s["y"].float(), s["x"].float()
    post, gate = _over(s["post"]), _over(s["gate"])
    un, ur = _normed(y, c["center"]) if c["post"] else (y, None)
    u = _affine(un, post, _over(s["post_bias"])) if c["post"] else y
    h = x + c["scale"] * (u if gate is None else gate * u)
    hn, hr = _normed(h, c["center"])
    z = _affine(hn, _over(s["weight"]), _over(s["weight_bias"]))
    return h, z, (u, un, ur, hn, hr)


def _norm_grad(dv, vn, r, center):
    """Gradient of normalised rows: dv is the one of vn."""
    dv = dv - dv.mean(-1, keepdim=True) if center else dv
    return r * (dv - vn * (dv * vn).mean(-1, keepdim=True))


def _plain_train(s):
    c = s["c"]
    h, z, (u, un, ur, hn, hr) = _plain_norm(s)
    dz, rows = s["dz"].float(), (1, 2)
    gate = _over(s["gate"])
    dx = s["dh"].float() + _norm_grad(dz * _over(s["weight"]), hn, hr, c["center"])
    g = {"x": dx, "weight": (dz * hn).sum(rows), "weight_bias": dz.sum(rows)}
    du = c["scale"] * dx
    if gate is not None:
        of_rows = du * u
        g["gate"] = of_rows if c["gate"] == "token" else of_rows.sum((1, 2) if c["gate"] == "model" else 2)
        du = du * gate
    g["y"] = du
    if c["post"]:
        g["post"], g["post_bias"] = (du * un).sum(rows), du.sum(rows)
        g["y"] = _norm_grad(du * _over(s["post"]), un, ur, c["center"])
    dt = TYPES[c["dtype"]]
    return [h.to(dt), z.to(dt)] + [g[k].to(dt) for k in _INPUTS if s[k] is not None]


def _plain_codes(x):
    """Rows as whole numbers up to 127 (in 32 bits) and their scales."""
    top = x.abs().amax(-1, keepdim=True).clamp(min=FLOOR)
    scale = top / torch.full_like(top, 127.0)              # by a tensor: by a number it is a product with 1 / number
    return torch.round(x / scale), scale


def _plain_linear(codes, scale, layer, act="none", wide=torch.float32):
    w, ws, bias = layer
    n = w.shape[0]
    acc = torch.matmul(codes.flatten(1, 2).to(wide), w.to(wide).transpose(1, 2)).view(*codes.shape[:3], -1)
    y = acc * scale * ws.view(n, 1, 1, -1)
    y = y if bias is None else y + bias.float().view(n, 1, 1, -1)
    if act == "relu":
        y = y.clamp(min=0)
    elif act == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y


def _plain(s):
    c, dt = s["c"], TYPES[s["c"]["dtype"]]
    if c["kind"] == "train":
        return _plain_train(s)
    if c["kind"] == "linear8":
        wide = torch.float64 if dt == torch.float32 else torch.float32     # sums of codes pass 2 ** 24
        return _plain_linear(*_plain_codes(s["x"].float()), s["layer"], c["act"], wide).to(dt)
    h, z, _ = _plain_norm(s)
    if c["kind"] == "norm":
        return h.to(dt), z.to(dt)
    if c["kind"] == "proj8":
        return h.to(dt), _plain_linear(*_plain_codes(z), s["layer"]).to(dt)
    a = _plain_linear(*_plain_codes(z), s["up"], "gelu").to(dt)
    return h.to(dt), a, _plain_linear(*_plain_codes(a.float()), s["down"]).to(dt)


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------

def _package():
    import os
    import sys
    at = os.path.join(os.getcwd(), "pytorch-parallel-compiler_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import wide_compiler
    return wide_compiler


def _calls(s):
    ops, c = _package().ops, s["c"]
    dt = TYPES[c["dtype"]]
    acts = {"none": ops.ACT_NONE, "relu": ops.ACT_RELU, "gelu": ops.ACT_GELU}
    if c["kind"] == "linear8":
        w, ws, bias = s["layer"]
        codes, scale = ops.quantize_rows(s["x"])
        return ops.linear_int8(codes, scale, w, ws, bias, acts[c["act"]], dtype=dt)
    args = (s["x"], s["y"], s["weight"])
    kw = dict(bias=s["weight_bias"], post_weight=s["post"], post_bias=s["post_bias"], gate=s["gate"],
              scale=c["scale"], eps=EPS, center=c["center"])
    if c["kind"] in ("norm", "train"):
        h, z = ops.residual_norm(*args, **kw)
        if c["kind"] == "norm":
            return h, z
        grads = torch.autograd.grad((h, z), [s[k] for k in _INPUTS if s[k] is not None], (s["dh"], s["dz"]))
        return [h.detach(), z.detach(), *grads]
    h, codes, scale = ops.residual_norm_quantize(*args, **kw)
    if c["kind"] == "proj8":
        w, ws, bias = s["layer"]
        return h, ops.linear_int8(codes, scale, w, ws, bias, dtype=dt)
    w, ws, bias = s["up"]
    a = ops.linear_int8(codes, scale, w, ws, bias, ops.ACT_GELU, dtype=dt)
    w, ws, bias = s["down"]
    return h, a, ops.linear_int8(*ops.quantize_rows(a), w, ws, bias, dtype=dt)


def run(state):
    if own:
        return _calls(state)
    with torch.no_grad():
        return _plain(state)


def work(case):
    c, e = case, SIZE[case["dtype"]]
    m = c["n"] * c["b"] * c["t"]
    k = c.get("k", c.get("d"))
    product = lambda o, k, bias: {  # noqa: E731
        "bytes": c["n"] * o * (k + 4 + (e if bias else 0)), "flops": 2 * m * o * k}
    if c["kind"] == "linear8":
        p = product(c["o"], k, c["bias"])
        return {"bytes": p["bytes"] + m * (k + c["o"]) * e, "flops": p["flops"] + 4 * m * k}
    params = c["n"] * k * (1 + c["post"]) * (1 + c["center"])
    if c["gate"] != "none":
        params += math.prod(_gate_shape(c))
    if c["kind"] == "train":
        # x, y, dh, dz read; h, z, dx, dy written; the parameters read and their gradients written
        return {"bytes": (8 * m * k + 2 * params) * e, "flops": 40 * m * k}
    norm = {"bytes": (3 * m * k + params) * e, "flops": 15 * m * k}        # x and y read, h written
    if c["kind"] == "norm":
        return {"bytes": norm["bytes"] + m * k * e, "flops": norm["flops"]}
    up = product(c["o"], k, c["bias"])
    bytes_, flops = norm["bytes"] + up["bytes"] + m * c["o"] * e, norm["flops"] + up["flops"]
    if c["kind"] == "mlp8":
        down = product(k, c["o"], c["bias"])
        bytes_, flops = bytes_ + down["bytes"] + m * k * e, flops + down["flops"]
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c, dt = s["c"], TYPES[case["dtype"]]

    def norm(v, w, b):
        var, mean = torch.var_mean(v, -1, correction=0, keepdim=True)
        if not c["center"]:
            var, mean = var + mean * mean, torch.zeros_like(mean)
        out = (v - mean) / torch.sqrt(var + EPS) * w.view(c["n"], 1, 1, -1)
        return out if b is None else out + b.view(c["n"], 1, 1, -1)

    def held(v):
        """The values that the codes of these rows stand for (a scale and the
        quotient that is rounded are 32-bit numbers), without the scale."""
        scale = (v.abs().amax(-1, keepdim=True).clamp(min=FLOOR) / 127).float().double()
        return torch.round((v / scale).float().double()), scale

    def product(rows, layer, act="none"):
        (codes, scale), (w, ws, bias) = rows, layer
        out = torch.einsum("nbtk,nok->nbto", codes, w.double()) * scale * ws.double()[:, None, None]
        out = out if bias is None else out + bias.double()[:, None, None]
        return {"none": lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu}[act](out)

    if c["kind"] == "linear8":
        return product(held(s["x"].double()), s["layer"], c["act"])
    p = {k: None if s[k] is None else s[k].detach().double().requires_grad_(c["kind"] == "train") for k in _INPUTS}
    u = norm(p["y"], p["post"], p["post_bias"]) if c["post"] else p["y"]
    if p["gate"] is not None:
        u = u * p["gate"].reshape(p["gate"].shape[:-1] + (1,) * (4 - p["gate"].dim()) + (c["d"],))
    h = p["x"] + c["scale"] * u
    z = norm(h, p["weight"], p["weight_bias"])
    if c["kind"] == "norm":
        return h, z
    if c["kind"] == "train":
        grads = torch.autograd.grad((h, z), [v for v in p.values() if v is not None],
                                    (s["dh"].double(), s["dz"].double()))
        return [h.detach(), z.detach(), *grads]
    if c["kind"] == "proj8":
        return h, product(held(z), s["layer"])
    a = product(held(z), s["up"], "gelu")
    return h, a, product(held(a.to(dt).double()), s["down"])
