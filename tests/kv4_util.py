"""The 4-bit cache's format and attention over it, written from their definitions in numpy: levels in 32 bits (the definition's own), everything else in 64."""
import numpy as np

PAGE = 128


def quantise(x):
    """codes, lo, step of x [..][head_dim] (float32), groups of 64 channels; a group with a number that is not finite: codes 0, lo NaN, step 0"""
    f = np.float32
    with np.errstate(all="ignore"):
        g = np.ascontiguousarray(x, f).reshape(*x.shape[:-1], -1, 64)
        low = g.min(-1, keepdims=True)
        b = low.view(np.uint32).astype(np.uint64)
        lo = (np.where(low < 0, b + 0xFFFF, b) & 0xFFFF0000).astype(np.uint32).view(f)
        spread = (g.max(-1, keepdims=True) - lo).astype(f)
        step = (((spread * f(1.0 / 15.0)).astype(f).view(np.uint32).astype(np.uint64) + 0xFFFF) & 0xFFFF0000).astype(np.uint32).view(f)
        step = np.maximum(step, f(2.0 ** -126))
        n = np.minimum(np.rint((g - lo).astype(f) * (f(1) / step).astype(f)), f(15))
    fine = np.isfinite(g).all(-1, keepdims=True) & np.isfinite(spread)
    return np.where(fine, n, 0).reshape(x.shape), np.where(fine, lo, f(np.nan))[..., 0], np.where(fine, step, f(0))[..., 0]


def values(x):
    """what a cache gives back for x, in 64 bits, and how large the numbers are that its products go through (|lo| + 143 step)"""
    n, lo, step = quantise(x)
    lo, step = (np.repeat(a.astype(np.float64), 64, -1) for a in (lo, step))
    return lo + step * n, np.abs(lo) + 143 * step


def attend(q, k, v, pos, window=0, scale=None, big=None):
    """softmax(scale q k^T) v of queries [T][heads][D] at positions pos over keys and values [n][kv_heads][D], 64 bits; a row that sees nothing: zeros.
    big = (keys' sizes, values' sizes): also per output a bound on the sizes that go into its score (the largest) and into it"""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    T, H, D = q.shape
    G = H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, s_size, o_size = np.zeros((T, H, D)), np.zeros((T, H, 1)), np.zeros((T, H, D))
    for i in range(T):
        lo, hi = max(0, pos[i] - window + 1) if window else 0, min(len(k), pos[i] + 1)
        if hi <= lo:
            continue
        for h in range(H):
            s = scale * (k[lo:hi, h // G] @ q[i, h])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ v[lo:hi, h // G]
            if big is not None:
                s_size[i, h] = abs(scale) * (big[0][lo:hi, h // G] @ np.abs(q[i, h])).max()
                o_size[i, h] = p @ big[1][lo:hi, h // G]
    return (out, s_size, o_size) if big is not None else out


def bound(out, s_size, o_size, keys, eps, terms):
    """How far an output may be from 64 bits: half a step of its type (eps) of the value; a score of sizes S is off by (2 D + 24) roundings of 2^-24 of them (two chained
    products of 128, the factors, the scale) and, of queries in two 16-bit terms, by 2^-17; an exponential's relative error is its argument's plus 2^-22; a weight is
    two 16-bit terms (2^-17) or one (2^-9); a sum of n numbers is off by n 2^-24 of their sizes.  Both numerator and denominator carry the exponentials' errors."""
    D = out.shape[-1]
    score = s_size * ((2 * D + 24) * 2.0 ** -24 + (2.0 ** -17 if terms == 2 else 0)) + 2.0 ** -22
    weight = 2.0 ** -17 if terms == 2 else 2.0 ** -9
    return 0.5 * eps * np.abs(out) * 1.01 + o_size * (2 * score + weight + (keys + 64) * 2.0 ** -24) + 1e-30
