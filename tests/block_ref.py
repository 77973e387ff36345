"""64-bit formulas of the block-boundary operators with bounds on what fp32
arithmetic makes of them.

U = 2^-24 is half a step of fp32 at 1. A sum over a row is taken as up to 32
values in a chain in a thread, then two trees of at most 5 levels: it is off by
at most 42 U times the sum of magnitudes.

Normalised rows vn = (v - m) r, with a = mean |v| and kappa = (rms(v) + a) / rms(v - m)
(1 for an RMS norm): m is off by 43 U a, so v - m by U (43 a + 2 |v|), the sum of
squares relatively by 2 U (45 kappa) + 45 U, r by half of that and 3 U, so

    |error of vn| <= eps (1 + |vn|),  eps = U (50 kappa + 40).

An error dv that the values already carry adds r (dv + mean dv) + |vn| r rms(dv).

Gradient t = r (g - vn c1 - c2) with c1 = mean(g vn), c2 = mean(g): with the
errors of vn, r (eps, relative) and of the sums (45 U <= eps / 2),

    |error| <= 4 eps r (|g| + (1 + |vn|) mean(|g| (1 + |vn|)))

and an error dg of g adds r (dg + (1 + |vn|) mean(dg (1 + |vn|))).

Sums over R rows are chains of at most R + 64 additions.
"""
import torch

U = 2.0 ** -24


def half_ulp(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step of the smallest numbers."""
    f = torch.finfo(dtype)
    return f.tiny * f.eps / 2


def rounded(value, err, dtype):
    """Bound of a result that is stored in dtype."""
    return err + half_ulp(dtype) * (value.abs() + err) + tiny(dtype)


def over(p, x):
    """[N, D] or a gate's shape over the rows of x [N, ..., D], in 64 bits."""
    return p.double().view(p.shape[:-1] + (1,) * (x.dim() - p.dim()) + p.shape[-1:])


class Norm:
    """Normalised rows of v (whose values are off by dv), their factor, bounds."""

    def __init__(self, v, dv, eps, center):
        mean = lambda t: t.mean(-1, keepdim=True)
        rms = lambda t: t.square().mean(-1, keepdim=True).sqrt()
        vc = v - mean(v) if center else v
        self.r = (mean(vc * vc) + eps).rsqrt()
        self.vn = vc * self.r
        kappa = torch.ones_like(self.r)
        if center:
            # with eps under the root a row of equal values is no worse than rms = sqrt(eps)
            kappa = (rms(v) + mean(v.abs())) * self.r
        self.eps = U * (50 * kappa + 40) + self.r * (rms(dv) + mean(dv))
        self.err = self.eps * (1 + self.vn.abs()) + self.r * dv

    def grad(self, g, dg, center):
        mean = lambda t: t.mean(-1, keepdim=True)
        t = self.r * (g - self.vn * mean(g * self.vn) - (mean(g) if center else 0))
        one = 1 + self.vn.abs()
        rel = (self.err / one).amax(-1, keepdim=True)
        err = 4 * rel * self.r * (g.abs() + one * mean(g.abs() * one)) + self.r * (dg + one * mean(dg * one))
        return t, err


def residual_norm(x, y, weight, bias=None, post_weight=None, post_bias=None, gate=None, scale=1.0, eps=1e-6,
                  center=False, dh=None, dz=None):
    """{name: (value, bound)} of h and z, and of the gradients where dh, dz are
    given. Values as they come out in x's dtype, z also ("z32") before rounding."""
    dtype, xd = x.dtype, x.double()
    zero = torch.zeros_like(xd)
    scale = float(torch.tensor(scale, dtype=torch.float32))
    eps = float(torch.tensor(eps, dtype=torch.float32))
    w, b = over(weight, x), zero if bias is None else over(bias, x)
    out, un = {}, None
    if y is None:
        u = du = zero
        g = torch.zeros(1, dtype=torch.float64)
    else:
        g = torch.ones(1, dtype=torch.float64) if gate is None else over(gate, x)
        if post_weight is None:
            u, du = y.double(), zero
        else:
            un = Norm(y.double(), zero, eps, center)
            pw, pb = over(post_weight, x), zero if post_bias is None else over(post_bias, x)
            u = un.vn * pw + pb
            du = un.err * pw.abs() + 2 * U * ((un.vn * pw).abs() + pb.abs())
    # the weights are folded, h = un (scale g pw) + (x + scale g pb): two roundings
    # of each product of weights, one each of the sum and of the last step
    k = scale * g
    h = xd + k * u
    amp = u.abs() if un is None else (un.vn * pw).abs() + pb.abs()
    eh = k.abs() * du + 4 * U * (k.abs() * amp + xd.abs())
    hn = Norm(h, eh if y is not None else zero, eps, center)
    z = hn.vn * w + b
    ez = hn.err * w.abs() + 2 * U * ((hn.vn * w).abs() + b.abs())
    out["h"] = (h, rounded(h, eh, dtype))
    out["z"] = (z, rounded(z, ez, dtype))
    out["z32"] = (z, ez)
    if dh is None and dz is None:
        return out
    dh = zero if dh is None else dh.double()
    dz = zero if dz is None else dz.double()
    model = tuple(range(1, x.dim() - 1))

    def summed(name, terms, errs, dims):
        rows = 1
        for i in dims:
            rows *= terms.shape[i]
        total = terms.sum(dims) if dims else terms
        err = errs + (rows + 64) * U * terms.abs() + 4 * U * errs
        out[name] = (total, rounded(total, err.sum(dims) if dims else err, dtype))

    t, et = hn.grad(dz * w, U * (dz * w).abs(), center)
    dx, ex = dh + t, et + 2 * U * (dh.abs() + t.abs())
    out["dx"] = (dx, rounded(dx, ex, dtype))
    summed("dweight", dz * hn.vn, dz.abs() * hn.err + U * (dz * hn.vn).abs(), model)
    if bias is not None:
        summed("dbias", dz, zero, model)
    if y is None:
        return out
    ds, es = k * dx, k.abs() * ex + 3 * U * (k * dx).abs()
    if gate is not None:
        dims = tuple(range(gate.dim() - 1, x.dim() - 1))
        terms = scale * dx * u
        summed("dgate", terms, abs(scale) * (amp * ex + dx.abs() * du) + 6 * U * abs(scale) * dx.abs() * amp, dims)
        if dims and un is not None:              # pw A + pb B: two sums that may cancel
            v, e = out["dgate"]
            rows = terms[0].numel() // terms.shape[-1]
            out["dgate"] = (v, e + (rows + 66) * U * (abs(scale) * dx.abs() * amp).sum(dims))
    if un is None:
        out["dy"] = (ds, rounded(ds, es, dtype))
        return out
    summed("dpost_weight", ds * un.vn, es * un.vn.abs() + ds.abs() * un.err + U * (ds * un.vn).abs(), model)
    if post_bias is not None:
        summed("dpost_bias", ds, es, model)
    t, et = un.grad(ds * pw, es * pw.abs() + U * (ds * pw).abs(), center)
    out["dy"] = (t, rounded(t, et, dtype))
    return out


def codes(z, ez):
    """Bounds of the codes of fp32 rows that are off by ez: (scale, its bound,
    quotient, its bound). A code is the quotient rounded: half a step more.
    The quotient's bound divides by the least that the scale may be, scale - es;
    where that is not positive (one channel under a LayerNorm: z is all
    cancellation), code and quotient, both within 127, are at most 254 apart."""
    top = z.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -40)
    scale = top / 127
    es = ez.amax(-1, keepdim=True) / 127 + U * scale
    q = z / scale
    least = scale - es
    eq = torch.where(least > 0, (ez + q.abs() * es) / least + U * q.abs(), torch.full_like(q, 254.0))
    return scale.squeeze(-1), es.squeeze(-1), q, eq


def assert_within(got, want, bound, what=""):
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values outside their bounds; worst "
                           f"{float((off / bound)[bad].max()) if bad.any() else 0:.3g} times, first at "
                           f"{bad.nonzero()[0].tolist()}: {float(got[bad][0])} for {float(want[bad][0])}")
