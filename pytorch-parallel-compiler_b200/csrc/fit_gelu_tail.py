"""Coefficients of the GELU of linear_int8.cu's 16-bit results.

gelu(x) = max(x, 0) - a Q(a) with a = |x| and Q(a) = erfc(a / sqrt 2) / 2, the
tail of the normal distribution. log2 Q(a) = -a^2 log2(e) / 2 + r(a), and r, which
is smooth, is fitted by a polynomial of degree 8 on [0, 8]: least squares at
Chebyshev nodes, the weights raised where the error is large until it is even.
Prints the coefficients (lowest power first) and the largest relative error of Q
with them, in 64 bits.
"""
import math

import numpy as np

DEGREE, END = 8, 8.0


def tail_log2(a):
    """r(a): log2 of erfcx(a / sqrt 2) / 2, erfcx by its continued fraction (Lentz
    form run backwards) past 2, by erfc before."""
    out = np.empty_like(a)
    for i, v in enumerate(a / math.sqrt(2)):
        if v < 2:
            e = math.erfc(v) * math.exp(v * v)
        else:
            f = 0.0
            for k in range(200, 0, -1):
                f = (k / 2) / (v + f)
            e = 1 / (math.sqrt(math.pi) * (v + f))
        out[i] = math.log2(e / 2)
    return out


def fit():
    nodes = (np.cos(np.pi * (np.arange(2000) + 0.5) / 2000) + 1) * END / 2
    basis = np.polynomial.chebyshev.chebvander(2 * nodes / END - 1, DEGREE)
    want, weight, best = tail_log2(nodes), np.ones_like(nodes), (np.inf, None)
    for _ in range(400):
        c = np.linalg.lstsq(basis * np.sqrt(weight)[:, None], want * np.sqrt(weight), rcond=None)[0]
        off = np.abs(basis @ c - want)
        if off.max() < best[0]:
            best = off.max(), c
        weight = weight * (off / off.max() + 1e-3) ** 0.3
        weight /= weight.mean()
    poly = np.polynomial.chebyshev.Chebyshev(best[1], domain=[0, END]).convert(kind=np.polynomial.Polynomial)
    return poly.coef, best[0] * math.log(2)


if __name__ == "__main__":
    coef, err = fit()
    print(", ".join(f"{np.float32(c)!r}" for c in coef))
    print(f"relative error of Q: {err:.2e}")
