"""The limits of kv4_near.py, on the CPU: what the operators are to give passes them, in 32-bit arithmetic too, and what a wrong kernel would give does not."""
import numpy as np
import pytest

from kv4_near import PORTIONS, TOKENS, Held, attend, inputs, queries, rounded, weights, why_not


def bf16(x):
    return rounded(x, "bf16")


def terms(x, n):
    """x as the sum of n terms of 8 bits each, to nearest"""
    out = np.zeros_like(x)
    for _ in range(n):
        out = out + bf16(x - out)
    return out


def altered(q, k, v, pos, what):
    """outputs in 64 bits of an evaluation that is not the operators'"""
    T, H, D = q.shape
    G, j = H // k.x.shape[1], np.arange(len(k.x))
    out = np.zeros((T, H, D))
    seen = {"own": j != pos[0], "block": (j > pos[0]) | (j // 32 != pos[0] // 32), "first": j > 0}.get(what)
    for t in range(T):
        for h in range(k.x.shape[1]):
            hs = slice(h * G, h * G + G)
            kk, vv, qq = k.x[:, h], v.x[:, h], q[t, hs].astype(np.float64)
            if what == "all bf16":
                kk, vv, qq = bf16(kk), bf16(vv), bf16(qq)
            if what == "two query terms":
                qq = terms(qq, 2)
            if what == "uniform":
                qq = qq * 0
            p, _ = weights(qq, Held.of(kk), 0, pos[t], 0, D ** -0.5, seen)
            if what == "all bf16":
                p = bf16(p / p.max(-1, keepdims=True))
                p = p / p.sum(-1, keepdims=True)
            if what in ("one weight term", "two weight terms"):
                n = 1 if what == "one weight term" else 2
                m = p.max(-1, keepdims=True)
                step = np.repeat(v.step[:, h], 64, -1)
                base = np.repeat(v.lo[:, h], 64, -1) + (7.5 * step if n == 2 else 0)
                codes = v.n[:, h] - (7.5 if n == 2 else 0)
                for g in range(D // 64):
                    c = slice(64 * g, 64 * g + 64)
                    w = terms(p / m * v.step[:, h, g], n) * m
                    out[t, hs, c] = w @ codes[:, c] + p @ base[:, c]
                continue
            out[t, hs] = p @ vv + (0.2 if what == "shifted" else 0)
    return out * (0 if what == "zeros" else 1)


class _Of(Held):
    def __init__(self, x):
        self.x = x[:, None]
        self.n, self.lo, self.step = self.x * 0, np.zeros((len(x), 1, x.shape[1] // 64)), np.zeros((len(x), 1, x.shape[1] // 64))


Held.of = staticmethod(_Of)


def in_32_bits(q, k, v, pos):
    f = np.float32
    T, H, D = q.shape
    G = H // k.x.shape[1]
    out = np.zeros((T, H, D))
    for t in range(T):
        for h in range(k.x.shape[1]):
            hs, n = slice(h * G, h * G + G), pos[t] + 1
            s = (q[t, hs].astype(f) @ k.x[:n, h].astype(f).T) * f(D ** -0.5)
            p = np.exp(s - s.max(-1, keepdims=True))
            out[t, hs] = (p @ v.x[:n, h].astype(f)) / p.sum(-1, keepdims=True, dtype=f)
    return out


def cases():
    for lens, group, kv in TOKENS:
        for n in sorted(set(lens)):
            yield n, [n - 1], group, kv
    for lens, counts, group in PORTIONS:
        for n, c in sorted(set(zip(lens, counts))):
            yield n, sorted({n - c, n - 1}), group, 2


WRONG = ["zeros", "uniform", "own", "block", "first", "shifted", "all bf16", "one weight term"]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hd", [64, 128])
def test_wrong_outputs_are_told_from_right_ones(hd, dtype):
    """for every length, group and type that the operators are tested with: the right values rounded to the type pass, and 32-bit sums do; outputs of zero, uniform weights, a token's own
    key left out, its block of 32, or the sequence's first token (each where the weight that is missing is 1e-3 of all or more), values off by 0.2, everything in bf16, weights in one
    16-bit term do not"""
    for n, pos, group, kv in cases():
        k, v = (Held(x) for x in inputs([n], kv, hd, dtype, n + hd))
        q = queries(len(pos), kv * group, hd, dtype, 9, 1.5).astype(np.float64)
        want, size = attend(q, k, v, pos)
        assert why_not(rounded(want, dtype), want, size, n, dtype) is None
        assert why_not(rounded(in_32_bits(q, k, v, pos), dtype), want, size, n, dtype) is None, (n, pos)
        for what in WRONG:
            p = np.stack([weights(q[0, h * group:h * group + group], k, h, pos[0], 0, hd ** -0.5)[0] for h in range(kv)])
            j = np.arange(n)
            lost = {"own": p[..., j == pos[0]], "block": p[..., (j <= pos[0]) & (j // 32 == pos[0] // 32)], "first": p[..., :1]}.get(what)
            if pos[0] == 0 and what not in ("zeros", "shifted") or lost is not None and lost.sum(-1).max() < 1e-3:
                continue
            if what in ("all bf16", "one weight term") and pos[0] < 4 and dtype != "fp32":
                continue      # (the values of one or two tokens may be their own roundings)
            got = rounded(altered(q, k, v, pos, what), dtype)
            assert why_not(got, want, size, n, dtype) is not None, (what, n, pos, group)


def test_three_terms_are_told_from_two():
    """32-bit outputs: test_hip_kv4_values.test_32_bit_outputs_have_three_terms, whose limit of 20 steps of 2^-24 two terms of a query or of a weight do not meet and 32-bit sums do"""
    for n, hd in [(700, 64), (4096, 128)]:
        k, v = (Held(x) for x in inputs([n], 1, hd, "fp32", n))
        q = queries(1, 32, hd, "fp32", 5).astype(np.float64)
        want, _ = attend(q, k, v, [n - 1])

        def off(x):
            return np.sqrt(((rounded(x, "fp32") - want) ** 2).sum() / (want ** 2).sum())
        assert off(in_32_bits(q, k, v, [n - 1])) < 20 * 2.0 ** -24
        for what in ("two weight terms", "two query terms"):
            assert off(altered(q, k, v, [n - 1], what)) > 1.5 * 20 * 2.0 ** -24, what


def test_the_limits_of_kv4_util_hold_less():
    """bound() of kv4_util.py, with which test_hip_kv4.py goes on: outputs of zero are within it for 713 tokens, and outside of why_not"""
    from kv4_util import attend as attend_, bound, values
    kx, vx = inputs([713], 1, 64, "fp32", 1)
    q = queries(1, 4, 64, "fp32", 9, 1.5)
    (k, kb), (v, vb) = values(kx), values(vx)
    want, s, o = attend_(q, k, v, [712], big=(kb, vb))
    assert (np.abs(want) <= bound(want, s, o, 713, 2.0 ** -23, 2)).all()
    right, size = attend(q.astype(np.float64), Held(kx), Held(vx), [712])
    assert np.allclose(right, want, rtol=1e-12, atol=1e-14)
    assert why_not(want * 0, right, size, 713, "fp32") is not None
