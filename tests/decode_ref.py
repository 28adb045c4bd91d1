"""Plain f64 statements of the decode-step operators, and the numbers that their tests' tolerances come from.

Rounding model.  q, x and the softmax weights enter the tensor cores as two f16 parts: half a step of 22 bits, 2^-23
relative, and products with codes are exact.  A block's 64 products (two parts of 32 values) are added in f32, some
sqrt(64) steps of 2^-23 of the largest partial sum, then the blocks: together at most 2^-20 of sum |a||b| per dot
product.  Sums over tokens: at most 2 L / 4 additions per warp, sqrt(1000) * 2^-23 = 2^-18 of sum p|v| for L <= 2000.
"""
import numpy as np

import vortx_b200 as vb

DOT = 2.0 ** -20
SUM = 2.0 ** -18


def quantised(qt, a):
    """The values that a's codes stand for, in f64; blocks along the last axis."""
    a = np.ascontiguousarray(a, np.float32)
    flat = a.reshape(-1, a.shape[-1])
    return vb.dequantize_host(qt, vb.quantize(qt, flat), *flat.shape).astype(np.float64).reshape(a.shape)


def attention(q, k, v, may, scale):
    """q [n, D], k, v [L, D], may [n, L]; the result and how far f32 sums may be from it."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    with np.errstate(invalid="ignore", over="ignore"):
        s = np.where(may, scale * q @ k.T, -np.inf)
    out, tol = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1]))
    for i in range(len(q)):
        at = may[i]
        if at.any():
            p = np.exp(s[i, at] - s[i, at].max())
            p /= p.sum()
            out[i] = p @ v[at]
            d = DOT * abs(scale) * (np.abs(q[i]) @ np.abs(k[at]).T).max()
            tol[i] = (2 * d + SUM) * (p @ np.abs(v[at]))
    return out, tol + 1e-30


def silu(a):
    return a / (1 + np.exp(-a))


def moe(x, router, gate, up, down, top_k, normalise):
    """x [T, H], gate / up [E, F, H], down [E, H, F] (f64 values); y, ids, weights, tolerance of y."""
    x, router = x.astype(np.float64), router.astype(np.float64)
    logits = x @ router.T
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :top_k]
    best = np.take_along_axis(logits, ids, 1)
    top = best[:, :1]
    weights = np.exp(best - top) / (np.exp(best - top) if normalise else np.exp(logits - top)).sum(1, keepdims=True)
    y, tol = np.zeros_like(x), np.zeros_like(x)
    # a logit's f32 sum: some sqrt(H / 32 + 5) steps, 2^-20 of sum |x||router|; a weight moves by twice that
    dw = 2 * DOT * (np.abs(x) @ np.abs(router).T).max(1)
    for t in range(len(x)):
        for j in range(top_k):
            e, w = ids[t, j], weights[t, j]
            g, u = gate[e] @ x[t], up[e] @ x[t]
            dg, du = (2 * DOT * (np.abs(m[e]) @ np.abs(x[t])) for m in (gate, up))
            h = silu(g) * u
            dh = 1.1 * dg * np.abs(u) + np.abs(silu(g)) * du + 2.0 ** -21 * np.abs(h)
            y[t] += w * (down[e] @ h)
            tol[t] += w * (np.abs(down[e]) @ (dh + 2 * DOT * np.abs(h)) + dw[t] * np.abs(down[e]) @ np.abs(h))
    return y, ids, weights, tol + 1e-30, dw
