"""What is measured of the decoder-attention operators of N fused models.

Four paths, each as its plain form (elementary torch operations in 32 bits)
and as the calls a user makes of ``wide_compiler``:

  rope    RMS norm of every query and key head, then the position rotation
  train   the same with its gradients (queries, keys and both norm weights)
  cache   a paged key-value cache: quantised as it is written, read back
  decode  attention of one new token over the paged cache
  step    one decoder step: norm + rotation + cache write, then the attention

Tensors are N-first: q [N, B, T, Hq, D], k and v [N, B, T, Hk, D] as views of
one fused projection, the cache [N, pages, Hk, page, D].
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "int8": torch.int8,
         "fp8": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "int8": 1, "fp8": 1}
CODE_MAX = {"int8": 127.0, "fp8": 448.0}
EPS = 1e-6
FLOOR = 2.0 ** -40          # smallest row maximum that an 8-bit row is scaled by


def listed():
    return [
        # prompts of several fused models, grouped key heads: the throughput case of the norm + rotation
        dict(name="rope_prompt_bf16", kind="rope", dtype="bf16", n=8, b=4, t=2048, hq=16, hk=4, d=128, rot=128,
             inter=False, pad=False),
        # one token for each sequence, as many key heads as query heads of 64: latency
        dict(name="rope_token_f16", kind="rope", dtype="f16", n=16, b=8, t=1, hq=8, hk=8, d=64, rot=64, inter=True,
             pad=False),
        # a training step of the norm + rotation, grouped key heads
        dict(name="train_bf16", kind="train", dtype="bf16", n=4, b=4, t=1024, hq=32, hk=8, d=128, rot=64, inter=False,
             pad=False),
        # odd sizes, part of the head rotated, padded rows, 32-bit gradients
        dict(name="train_f32_odd", kind="train", dtype="f32", n=3, b=5, t=77, hq=6, hk=2, d=84, rot=40, inter=True,
             pad=True),
        # prompts written to an 8-bit cache and read back (the context of a later piece of the prompt)
        dict(name="cache_int8_prompt", kind="cache", dtype="bf16", fmt="int8", n=8, b=4, t=4096, hk=8, d=128, page=64,
             pad=False),
        # padded prompts, pages of 24 tokens, heads of 72
        dict(name="cache_fp8_ragged", kind="cache", dtype="f16", fmt="fp8", n=2, b=7, t=333, hk=3, d=72, page=24,
             pad=True),
        # the first tokens of a chat: a short cache, as many key heads as query heads
        dict(name="decode_short_bf16", kind="decode", dtype="bf16", fmt="bf16", n=4, b=1, len=37, hq=8, hk=8, d=64,
             page=16, window=0, empty=False),
        # ordinary serving: a batch of ragged sequences for each model, grouped heads
        dict(name="decode_batch_bf16", kind="decode", dtype="bf16", fmt="bf16", n=8, b=16, len=4096, hq=32, hk=8,
             d=128, page=64, window=0, empty=False),
        # one sequence with a long context, 8-bit cache: the length has to be split
        dict(name="decode_long_int8", kind="decode", dtype="bf16", fmt="int8", n=1, b=1, len=131007, hq=16, hk=2,
             d=128, page=128, window=0, empty=False),
        # 32-bit models, heads of 84, pages that end inside a tile, a sliding window, sequences without tokens
        dict(name="decode_f32_window", kind="decode", dtype="f32", fmt="f32", n=2, b=9, len=1900, hq=6, hk=3, d=84,
             page=20, window=511, empty=True),
        # one decoder step of a large batch over a fp8 cache
        dict(name="step_fp8", kind="step", dtype="bf16", fmt="fp8", n=8, b=32, len=2048, hq=16, hk=4, d=128, rot=128,
             inter=False, page=64),
        # one decoder step of a small batch, heads of 64
        dict(name="step_bf16_small", kind="step", dtype="bf16", fmt="bf16", n=16, b=2, len=200, hq=8, hk=8, d=64,
             rot=64, inter=False, page=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _head(rng):
    """A head size: mostly the common ones, else any even size up to 256."""
    r = rng.random()
    if r < 0.5:
        return rng.choice((64, 96, 128, 256))
    if r < 0.85:
        return 8 * rng.randint(2, 32)
    return 2 * rng.randint(8, 128)


def draw(rng):
    kind = rng.choice(("rope", "train", "cache", "decode", "decode", "step"))
    d = _head(rng)
    hk = rng.choice((1, 2, 3, 4, 5, 8))
    group = rng.choice((1, 1, 2, 3, 4, 6, 8, 12, 16))
    rot = rng.choice((d, d, d // 2 // 2 * 2, d // 4 // 2 * 2 or 2))
    c = dict(kind=kind, dtype=rng.choice(("bf16", "bf16", "f16", "f32")), n=_log(rng, 1, 24), d=d, hk=hk)
    if kind in ("rope", "train"):
        c.update(b=_log(rng, 1, 16), t=_log(rng, 1, 4096), hq=hk * group, rot=rot, inter=rng.random() < 0.4,
                 pad=rng.random() < 0.3)
    elif kind == "cache":
        c.update(fmt=rng.choice(("int8", "fp8", c["dtype"])), b=_log(rng, 1, 16), t=_log(rng, 1, 4096),
                 page=_log(rng, 1, 256), pad=rng.random() < 0.3)
    else:
        c.update(fmt=rng.choice(("int8", "fp8", c["dtype"])), b=_log(rng, 1, 48), len=_log(rng, 1, 131072),
                 hq=hk * group, page=rng.choice((16, 32, 64, 128, _log(rng, 4, 256))))
        if kind == "decode":
            c.update(window=rng.choice((0, 0, 0, _log(rng, 1, 4096))), empty=rng.random() < 0.2)
        else:
            c.update(rot=rot, inter=rng.random() < 0.4)
            if c["dtype"] == "f32":      # a key rounded to 8 bits is read back in 16: a tie of its rounding is a whole code
                c["fmt"] = "f32"
    grow = [k for k in ("len", "t", "b", "n") if k in c]
    while work(c)["bytes"] > 6e8 or _held(c) > 4e8:
        k = max((g for g in grow if c[g] > 1), key=lambda g: c[g])
        c[k] = max(1, c[k] * 2 // 3)
    return c


def _held(c):
    """Values of the whole cache or of all heads (the plain form widens them)."""
    if "len" in c:
        return 2 * c["n"] * c["b"] * c["hk"] * (c["len"] + c["page"]) * c["d"]
    return c["n"] * c["b"] * c["t"] * (c.get("hq", 0) + 2 * c["hk"]) * c["d"]


# ---------------------------------------------------------------------------
# What a user's program has before the call
# ---------------------------------------------------------------------------

def _lengths(c):
    """[N, B] visible tokens of each sequence: ragged between half the longest
    and the longest; with ``empty``, every fourth has none."""
    i = torch.arange(c["n"] * c["b"]).view(c["n"], c["b"])
    ln = c["len"] - (i * 7919) % (c["len"] // 2 + 1)
    if c.get("empty"):
        ln = torch.where(i % 4 == 1, torch.zeros_like(ln), ln)
    return ln.to(torch.int32)


def _seen(c):
    ln = _lengths(c)
    w = c.get("window", 0)
    return int((ln.clamp(max=w) if w else ln).sum())


def _padded(c):
    """[B, T] True at padding rows: the tail of every second sequence."""
    t = torch.arange(c["t"])
    b = torch.arange(c["b"])
    keep = torch.where(b % 2 == 1, c["t"] - c["t"] // 3, torch.full_like(b, c["t"]))
    return (t[None, :] >= keep[:, None]) if c["pad"] else torch.zeros(c["b"], c["t"], dtype=torch.bool)


def _heads(c, t, g, dtype):
    """Views q, k, v of one fused projection [N, B, T, (Hq + 2 Hk) D]; a few
    channels are much larger than the rest, as trained projections have."""
    hq, hk, d = c.get("hq", 0), c["hk"], c["d"]
    x = torch.randn(c["n"], c["b"], t, hq + 2 * hk, d, device=DEV, generator=g, dtype=torch.float32)
    gain = torch.exp(0.5 * torch.randn(c["n"], 1, 1, hq + 2 * hk, d, device=DEV, generator=g))
    x = x.mul_(gain).to(dtype).view(c["n"], c["b"], t, -1)
    cut = lambda a, h: x[..., a * d:(a + h) * d].unflatten(-1, (h, d))  # noqa: E731
    return (cut(0, hq) if hq else None), cut(hq, hk), cut(hq + hk, hk)


def _tables(c, rows):
    i = torch.arange(0, c["rot"], 2, device=DEV, dtype=torch.float64) / c["rot"]
    ang = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * torch.pow(10000.0, -i)[None]
    return torch.cos(ang).float(), torch.sin(ang).float()


def _norm_weight(c, g, dtype):
    return (1 + 0.2 * torch.randn(c["n"], c["d"], device=DEV, generator=g)).to(dtype)


def _page_table(c, tokens, g):
    """[N, B, M] pages of each sequence in random order, and the pages held."""
    m = -(-tokens // c["page"])
    held = c["b"] * m + 2
    order = torch.rand(c["n"], held, device=DEV, generator=g).argsort(dim=1)
    return order[:, :c["b"] * m].reshape(c["n"], c["b"], m).to(torch.int32), held


def _pages(c, held, fmt, g):
    """One side of the cache as earlier steps left it: pages (and scales)."""
    shape = (c["n"], held, c["hk"], c["page"], c["d"])
    if fmt == "int8":
        x = torch.randint(-127, 128, shape, device=DEV, generator=g, dtype=torch.int8)
    elif fmt == "fp8":
        x = torch.randn(shape, device=DEV, generator=g, dtype=torch.float16).mul_(120).clamp_(-448, 448)
        return x.to(torch.float8_e4m3fn), torch.rand(shape[:4], device=DEV, generator=g) * 0.01 + 0.002
    else:
        return torch.randn(shape, device=DEV, generator=g, dtype=torch.float32).to(TYPES[fmt]), None
    return x, torch.rand(shape[:4], device=DEV, generator=g) * 0.03 + 0.005


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[c["dtype"]]
    s = dict(c=c)
    if c["kind"] in ("rope", "train", "step"):
        t = c.get("t", 1)
        s["q"], s["k"], s["v"] = _heads(c, t, g, dt)
        s["q_weight"], s["k_weight"] = _norm_weight(c, g, dt), _norm_weight(c, g, dt)
        if c["kind"] != "step":
            s["cos"], s["sin"] = _tables(c, t + 16)
            pos = torch.arange(t)[None, :] + (torch.arange(c["b"]) % 16)[:, None]
            s["positions"] = torch.where(_padded(c), torch.full_like(pos, -1), pos).to(DEV)
    if c["kind"] == "train":
        like = lambda x: torch.randn(x.shape, device=DEV, generator=g).to(dt)  # noqa: E731
        s["dq"], s["dk"] = like(s["q"]), like(s["k"])
        for name in ("q", "k", "q_weight", "k_weight"):
            s[name] = s[name].detach().requires_grad_(True)
    if c["kind"] == "cache":
        _, s["k"], s["v"] = _heads(c, c["t"], g, dt)
        s["table"], held = _page_table(c, c["t"], g)
        s["pages"] = _empty_pages(c, held)
        pos = torch.arange(c["t"]).expand(c["b"], -1)
        s["positions"] = torch.where(_padded(c), torch.full_like(pos, -1), pos).to(torch.int32).to(DEV)
    if c["kind"] in ("decode", "step"):
        s["lengths"] = _lengths(c).to(DEV)
        s["table"], held = _page_table(c, c["len"], g)
        k, ks = _pages(c, held, c["fmt"], g)
        v, vs = _pages(c, held, c["fmt"], g)
        s["pages"] = (k, v, ks, vs)
        if c["kind"] == "decode":
            s["q"] = torch.randn(c["n"], c["b"], c["hq"], c["d"], device=DEV, generator=g).to(dt)
            _unwritten(s)
        else:
            s["positions"] = (s["lengths"] - 1).unsqueeze(-1)
            s["cos"], s["sin"] = _tables(c, c["len"])
    return s


def _unwritten(s):
    """Slots that no token was written to hold anything: NaN here."""
    c, (k, v, ks, vs) = s["c"], s["pages"]
    t = torch.arange(s["table"].shape[2] * c["page"], device=DEV)
    n, b, t = torch.nonzero(t >= s["lengths"][..., None], as_tuple=True)
    page = s["table"].long()[n, b, t // c["page"]]
    for x in ((k, v) if ks is None else (ks, vs)):
        x[n, page, :, t % c["page"]] = float("nan")


def _empty_pages(c, held):
    shape = (c["n"], held, c["hk"], c["page"], c["d"])
    page = lambda: torch.zeros(shape, device=DEV, dtype=TYPES[c["fmt"]])  # noqa: E731
    scale = lambda: torch.zeros(shape[:4], device=DEV) if c["fmt"] in CODE_MAX else None  # noqa: E731
    return page(), page(), scale(), scale()


# ---------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------

def _rotate(u, co, si, inter, back=False):
    """The first 2*co.shape[-1] channels of u turned by the table's angles."""
    r = 2 * co.shape[-1]
    a, b = (u[..., 0:r:2], u[..., 1:r:2]) if inter else (u[..., :r // 2], u[..., r // 2:r])
    si = -si if back else si
    x, y = a * co - b * si, b * co + a * si
    turned = torch.stack((x, y), -1).flatten(-2) if inter else torch.cat((x, y), -1)
    return torch.cat((turned, u[..., r:]), -1)


def _table_rows(s):
    """cos, sin [.., B, T, 1, R/2] at the positions, and which rows count."""
    pos = s["positions"].long()
    at = pos.clamp(min=0)
    return s["cos"][at].unsqueeze(-2), s["sin"][at].unsqueeze(-2), (pos >= 0)[..., None, None]


def _plain_rope(s, x, w):
    co, si, keep = _table_rows(s)
    x = x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    y = _rotate(x * r * w.float()[:, None, None, None], co, si, s["c"]["inter"])
    return torch.where(keep, y, torch.zeros((), device=DEV))


def _plain_rope_grad(s, x, w, dy):
    co, si, keep = _table_rows(s)
    x, w = x.float(), w.float()[:, None, None, None]
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    du = torch.where(keep, _rotate(dy.float(), co, si, s["c"]["inter"], back=True), torch.zeros((), device=DEV))
    dw = (du * x * r).sum((1, 2, 3))
    gx = du * w
    return r * (gx - x * (r * r) * (gx * x).mean(-1, keepdim=True)), dw


def _plain_encode(x, fmt):
    """Rows as they are held: (codes, scales) in 8 bits, (rounded, None) else."""
    if fmt not in CODE_MAX:
        return x.to(TYPES[fmt]), None
    x = x.float()
    top = x.abs().amax(-1).clamp(min=FLOOR)
    scale = top / torch.full_like(top, CODE_MAX[fmt])      # by a tensor: by a number it is a product with 1 / number
    y = x / scale.unsqueeze(-1)
    return (torch.round(y) if fmt == "int8" else y).to(TYPES[fmt]), scale


def _bits(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _slots(s):
    """Page and offset of every position [N, B, T], and which rows count."""
    pos = s["positions"].long().expand(s["c"]["n"], s["c"]["b"], -1)
    at = pos.clamp(min=0)
    page = torch.gather(s["table"].long(), 2, at // s["c"]["page"])
    return page, at % s["c"]["page"], pos >= 0


def _plain_write(s, k, v):
    page, off, keep = _slots(s)
    n = torch.arange(s["c"]["n"], device=DEV)[:, None, None].expand_as(page)[keep]
    page, off = page[keep], off[keep]
    kp, vp, ks, vs = s["pages"]
    (kc, k1), (vc, v1) = _plain_encode(k, s["c"]["fmt"]), _plain_encode(v, s["c"]["fmt"])
    _bits(kp)[n, page, :, off] = _bits(kc)[keep]
    _bits(vp)[n, page, :, off] = _bits(vc)[keep]
    if ks is not None:
        ks[n, page, :, off] = k1[keep]
        vs[n, page, :, off] = v1[keep]


def _plain_read(s, dtype):
    page, off, keep = _slots(s)
    n = torch.arange(s["c"]["n"], device=DEV)[:, None, None]
    kp, vp, ks, vs = s["pages"]

    def one(x, scale):
        y = _bits(x)[n, page, :, off].view(x.dtype).float()
        y = y if scale is None else y * scale[n, page, :, off].unsqueeze(-1)
        return torch.where(keep[..., None, None], y, torch.zeros((), device=DEV)).to(dtype)

    return one(kp, ks), one(vp, vs)


def _plain_decode(s, q):
    c = s["c"]
    kp, vp, ks, vs = s["pages"]
    n, at = torch.arange(c["n"], device=DEV)[:, None, None], s["table"].long()
    tokens = at.shape[2] * c["page"]

    def wide(x, scale):
        y = _bits(x)[n, at].view(x.dtype).float()                      # [N, B, M, Hk, page, D]
        y = y if scale is None else y * scale[n, at].unsqueeze(-1)
        return y.transpose(2, 3).reshape(c["n"], c["b"], c["hk"], tokens, c["d"])

    t = torch.arange(tokens, device=DEV)
    ln = s["lengths"].long()[..., None]
    see = (t < ln) & ((t >= ln - c["window"]) if c.get("window") else True)
    see = see[:, :, None, None]
    q = q.float().unflatten(2, (c["hk"], -1))
    z = torch.matmul(q, wide(kp, ks).transpose(-1, -2)) / math.sqrt(c["d"])
    z = torch.where(see, z, torch.full((), -math.inf, device=DEV))
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    v = torch.where(see.transpose(-1, -2), wide(vp, vs), torch.zeros((), device=DEV))
    o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    return o.flatten(2, 3)


def _plain(s):
    c = s["c"]
    dt = TYPES[c["dtype"]]
    if c["kind"] in ("rope", "train"):
        out = [_plain_rope(s, s["q"], s["q_weight"]).to(dt), _plain_rope(s, s["k"], s["k_weight"]).to(dt)]
        if c["kind"] == "train":
            dq, dqw = _plain_rope_grad(s, s["q"], s["q_weight"], s["dq"])
            dk, dkw = _plain_rope_grad(s, s["k"], s["k_weight"], s["dk"])
            out += [dq.to(dt), dk.to(dt), dqw.to(dt), dkw.to(dt)]
        return out
    if c["kind"] == "cache":
        _plain_write(s, s["k"], s["v"])
        return _plain_read(s, dt)
    if c["kind"] == "decode":
        return _plain_decode(s, s["q"]).to(dt)
    q = _plain_rope(s, s["q"], s["q_weight"]).to(dt)
    _plain_write(s, _plain_rope(s, s["k"], s["k_weight"]), s["v"])
    k1, v1 = _plain_read(s, dt)
    return q, _plain_decode(s, q[:, :, 0]).to(dt), k1, v1


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
    wc = _package()
    ops, c = wc.ops, s["c"]
    if c["kind"] in ("decode", "step", "cache"):
        k, v, ks, vs = s["pages"]
        cache = wc.WidePagedCache(k, v, s["table"], k_scale=ks, v_scale=vs)
    if c["kind"] == "decode":
        return ops.decode_attention(s["q"], cache, s["lengths"], window=c["window"])
    if c["kind"] == "cache":
        ops.cache_write(cache, s["k"], s["v"], s["positions"])
        return ops.cache_read(cache, s["positions"], dtype=s["k"].dtype)
    rope = (s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"])
    if c["kind"] == "step":
        q = ops.qk_norm_rope_write(s["q"], s["k"], s["v"], *rope, cache, eps=EPS, interleaved=c["inter"])
        out = ops.decode_attention(q[:, :, 0], cache, s["lengths"])
        return (q, out, *ops.cache_read(cache, s["positions"], dtype=q.dtype))
    q, k = ops.qk_norm_rope(s["q"], s["k"], *rope, eps=EPS, interleaved=c["inter"])
    if c["kind"] == "rope":
        return [q, k]
    grads = torch.autograd.grad((q, k), (s["q"], s["k"], s["q_weight"], s["k_weight"]), (s["dq"], s["dk"]))
    return [q.detach(), k.detach(), *grads]


def run(state):
    if own:
        return _calls(state)
    with torch.no_grad():
        return _plain(state)


def work(case):
    c, e = case, SIZE[case["dtype"]]
    if c["kind"] in ("rope", "train"):
        rows = c["n"] * c["b"] * c["t"] * (c["hq"] + c["hk"])
        small = c["t"] * c["rot"] * 4 + c["b"] * c["t"] * 8 + 2 * c["n"] * c["d"] * e
        if c["kind"] == "rope":
            return {"bytes": 2 * rows * c["d"] * e + small, "flops": 8 * rows * c["d"]}
        return {"bytes": 5 * rows * c["d"] * e + small + 2 * c["n"] * c["d"] * e, "flops": 28 * rows * c["d"]}
    h = SIZE[c["fmt"]]
    row = c["d"] * h + (4 if c["fmt"] in CODE_MAX else 0)
    if c["kind"] == "cache":
        rows = 2 * c["n"] * int((~_padded(c)).sum()) * c["hk"]
        out = 2 * c["n"] * c["b"] * c["t"] * c["hk"] * c["d"] * e
        return {"bytes": rows * (c["d"] * e + 2 * row) + out + 4 * c["b"] * c["t"], "flops": 5 * rows * c["d"]}
    heads = c["n"] * c["b"] * c["hq"] * c["d"]
    read = 2 * _seen(c) * c["hk"]
    flops = 4 * _seen(c) * c["hq"] * c["d"]
    if c["kind"] == "decode":
        return {"bytes": read * row + 2 * heads * e, "flops": flops}
    new = c["n"] * c["b"] * c["hk"]
    return {"bytes": read * row + 3 * heads * e + 2 * new * (2 * c["d"] * e + row), "flops": flops}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]

    def turn(x, w):
        """Each pair of channels as a complex number times exp(i angle)."""
        x, w = x.double(), w.double()
        u = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["d"] + EPS) * w.view(c["n"], 1, 1, 1, c["d"])
        pos = s["positions"]
        r = c["rot"]
        e = torch.complex(s["cos"].double(), s["sin"].double())[pos.clamp(min=0).long()].unsqueeze(-2)
        h = u[..., :r].reshape(*u.shape[:-1], *((r // 2, 2) if c["inter"] else (2, r // 2)))
        h = h if c["inter"] else h.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(h.contiguous()) * e)
        z = z if c["inter"] else z.transpose(-1, -2)
        y = torch.cat((z.reshape(*u.shape[:-1], r), u[..., r:]), -1)
        return y * (pos >= 0).double()[..., None, None]

    def held(x):
        """The values that the cache holds for these rows."""
        if c["fmt"] not in CODE_MAX:
            return x.to(TYPES[c["fmt"]]).double()
        scale = (x.abs().amax(-1, keepdim=True).clamp(min=FLOOR) / CODE_MAX[c["fmt"]]).float().double()
        y = (x / scale).float().double()      # the quotient is a 32-bit number: it decides the ties
        if c["fmt"] == "int8":
            return torch.round(y) * scale
        step = torch.exp2((torch.frexp(y.abs()).exponent - 1).clamp(min=-6).double() - 3)
        return (torch.round(y / step) * step).clamp(-448, 448) * scale

    if c["kind"] in ("rope", "train"):
        ins = [s[k].detach().double().requires_grad_(c["kind"] == "train") for k in ("q", "k", "q_weight", "k_weight")]
        out = [turn(ins[0], ins[2]), turn(ins[1], ins[3])]
        if c["kind"] == "train":
            out += list(torch.autograd.grad(out, ins, [s["dq"].double(), s["dk"].double()]))
        return [x.detach() for x in out]
    if c["kind"] == "cache":
        keep = (s["positions"] >= 0).double()[..., None, None]
        return held(s["k"].double()) * keep, held(s["v"].double()) * keep

    q, new = s["q"], None
    if c["kind"] == "step":
        q1 = turn(s["q"], s["q_weight"])
        new = held(turn(s["k"], s["k_weight"])), held(s["v"].double())
        q = q1.to(TYPES[c["dtype"]])[:, :, 0]
    kp, vp, ks, vs = s["pages"]
    lengths = s["lengths"].cpu().tolist()
    o = torch.zeros(q.shape, device=DEV, dtype=torch.float64)
    for n in range(c["n"]):
        for b in range(c["b"]):
            ln = lengths[n][b]
            lo = max(0, ln - c["window"]) if c.get("window") else 0
            if ln == lo:
                continue
            pages = s["table"][n, b].long()[lo // c["page"]:-(-ln // c["page"])]
            first = lo // c["page"] * c["page"]
            side = []
            for x, scale in ((kp, ks), (vp, vs)):
                y = x[n].view(torch.uint8)[pages].view(x.dtype).double()
                y = y if scale is None else y * scale[n][pages].double().unsqueeze(-1)
                side.append(y.transpose(0, 1).reshape(c["hk"], -1, c["d"])[:, lo - first:ln - first].clone())
            if new is not None:
                side[0][:, -1], side[1][:, -1] = new[0][n, b, 0], new[1][n, b, 0]
            z = q[n, b].double().view(c["hk"], -1, c["d"]) @ side[0].transpose(1, 2) / c["d"] ** 0.5
            o[n, b] = (torch.softmax(z, -1) @ side[1]).reshape(c["hq"], c["d"])
    return o if new is None else (q1, o, new[0], new[1])
