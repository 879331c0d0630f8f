"""How near an output of attention over the 4-bit cache has to be to 64 bits: limits of the kernels' own errors, which zeros, uniform weights, a token left out or sums in fewer bits do not meet
(test_kv4_near.py holds them to that on the CPU)."""
import numpy as np

from kv4_util import quantise

STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}      # half a step of a type, relative to the value


def rounded(x, dtype):
    """64-bit numbers in an output's type, to nearest even, as 64-bit numbers"""
    if dtype == "bf16":
        m, e = np.frexp(x)
        return np.ldexp(np.rint(m * 256), e - 8)
    return np.asarray(x).astype(np.float16 if dtype == "fp16" else np.float32).astype(np.float64)


class Held:
    """what the cache holds for keys or values x [n][heads][D]: numbers, levels and codes in 64 bits"""

    def __init__(self, x):
        n, lo, step = quantise(x)
        self.n, self.lo, self.step = n.astype(np.float64), lo.astype(np.float64), step.astype(np.float64)
        self.x = np.repeat(self.lo, 64, -1) + np.repeat(self.step, 64, -1) * self.n


def weights(q, k, head, pos, window, scale, seen=None):
    """p [heads of one][n] of a token's queries q [heads of one][D] over key head `head`, and the score sizes: |scale| times, of every group, the lo's and the codes' part as they come out and, for what
    the codes' sum is on the way, the root of its terms' squares"""
    n = len(k.x)
    j = np.arange(n)
    see = (j <= pos) & ((j > pos - window) if window else True)
    if seen is not None:
        see = see & seen
    s = np.where(see, scale * (q @ np.where(see[:, None], k.x[:, head], 0).T), -np.inf)
    size = np.zeros(s.shape)
    for g in range(q.shape[-1] // 64):
        c = slice(64 * g, 64 * g + 64)
        size += np.abs(q[:, c].sum(-1)[:, None] * np.where(see, k.lo[:, head, g], 0)) + (np.abs(q[:, c] @ k.n[:, head, c].T) + np.sqrt(q[:, c] ** 2 @ (k.n[:, head, c] ** 2).T)) * np.where(see, k.step[:, head, g], 0)
    m = s.max(-1, keepdims=True)
    p = np.exp(s - np.where(np.isfinite(m), m, 0))
    return p / np.maximum(p.sum(-1, keepdims=True), 1e-300), abs(scale) * size


def attend(q, k, v, pos, window=0, scale=None, seen=None):
    """(outputs, largest score sizes by their weights) [T][heads][D], [T][heads] of queries q at positions pos over Held keys and values, in 64 bits; a row that sees nothing: zeros.
    seen: keys that are there at all"""
    q = np.asarray(q, np.float64)
    T, H, D = q.shape
    G = H // k.x.shape[1]
    out, size = np.zeros((T, H, D)), np.zeros((T, H))
    for t in range(T):
        for h in range(k.x.shape[1]):
            hs = slice(h * G, h * G + G)
            p, s = weights(q[t, hs], k, h, pos[t], window, D ** -0.5 if scale is None else scale, seen)
            out[t, hs] = p @ np.where((p > 0).any(0)[:, None], v.x[:, h], 0)
            size[t, hs] = np.sqrt((p * s * s).sum(-1))
    return out, size


def inputs(lens, kv_heads, hd, dtype, seed, scale=1.0):
    """keys and values [tokens of all sequences][kv_heads][hd] as the operators' tests take them: keys off zero by a channel's own, numbers of the storage type"""
    rng = np.random.default_rng(seed)
    off = 0.7 * rng.normal(size=(kv_heads, hd))
    k = scale * (rng.normal(size=(sum(lens), kv_heads, hd)) + off)
    v = scale * rng.normal(size=(sum(lens), kv_heads, hd))
    return tuple(rounded(x.astype(np.float32).astype(np.float64), dtype).astype(np.float32) for x in (k, v))


def queries(tokens, heads, hd, dtype, seed, scale=1.0):
    return rounded((scale * np.random.default_rng(seed).normal(size=(tokens, heads, hd))).astype(np.float32).astype(np.float64), dtype).astype(np.float32)


# (lengths, query heads a key / value head, key / value heads): a token of each sequence.  Behind `|` of the comment: walks that are divided between workgroups
TOKENS = [([1], 4, 1), ([2, 1, 33], 4, 1), ([127, 128, 129, 130], 1, 1), ([713], 4, 1), ([300, 5, 1000], 7, 1), ([64, 700], 16, 1), ([257, 31], 2, 1), ([513, 90], 3, 5), ([90, 400], 9, 2),
          ([3000], 4, 2), ([2100, 40], 8, 1), ([2500], 12, 1)]      # | the last line
# (lengths, tokens brought, query heads a key / value head), two key / value heads: few columns (16, 32) and more
PORTIONS = [([5], [5], 4), ([40, 3, 260], [2, 3, 5], 4), ([130, 700], [9, 8], 1), ([300], [300], 1), ([290, 33, 129], [70, 33, 1], 4), ([1000], [150], 7), ([200, 64], [17, 30], 16),
            ([2600], [3], 4), ([2200, 70], [7, 5], 4), ([3000], [40], 4)]      # | the last line


def own(size, keys, dtype):
    """How far a row (token, query head) may be from 64 bits beside the rounding of its output: rms over its channels relative to the row's rms.

    fp32, in units of 2^-24: a score is some ten roundings of its parts, which are as large as `size` and of either sign, so that they come to about 3 of them in quadrature, and a weight's
    relative error is its score's: 4 size.  Exponential, products, factors and the join 16.  A sum over n keys in blocks of 32 adds up n / 32 times: sqrt(n / 32) (three 16-bit terms of queries and weights
    leave 2^-24 and less).
    16 bits: weights of two 16-bit terms (2^-16 at most, 2^-18 in the rms) against codes up to 3.4 times as large as the values about their middle, and 16 blocks of two products' roundings in
    sums of such codes before the los join them, each some 2^-16: 2^-14 holds both twice over."""
    f32 = 2.0 ** -24 * (16 + 4 * size + np.sqrt(keys / 32))
    return f32 + (0 if dtype == "fp32" else 2.0 ** -14)


def why_not(out, want, size, keys, dtype):
    """None where outputs [T][heads][D] are as near to 64 bits as own() says, else what is wrong where.  A row's error is its own error and its rounding's, in quadrature: of the mean square that
    the rounding of the right values alone gives, no more than own() squared is left; and no channel is further off than half a step and ten own errors."""
    rms = np.sqrt((want ** 2).mean(-1))
    e = own(size, keys, dtype)
    rounding = ((rounded(want, dtype) - want) ** 2).mean(-1)
    got = ((out - want) ** 2).mean(-1)
    bad = ~(got <= 1.1 * rounding + (e * rms) ** 2)
    far = ~(np.abs(out - want) <= STEP[dtype] * np.abs(want) * 1.001 + (2.0 ** -25 if dtype == "fp16" else 0) + 10 * (e * rms)[..., None])
    if not bad.any() and not far.any():
        return None
    t = np.argwhere(bad) if bad.any() else np.argwhere(far)
    return f"{int(bad.sum())} rows, {int(far.sum())} channels; first {t[0].tolist()}: {np.sqrt(got.flat[0]):.3g}, largest {float(np.sqrt(np.nanmax(got / np.maximum(rms ** 2, 1e-300)))):.3g} of the row"
