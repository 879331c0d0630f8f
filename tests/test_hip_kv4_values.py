"""Values of attention over a 4-bit cache (tinygpt_amd.ops) near 64 bits, as near as kv4_near.py derives: short and long walks, divided and whole, every form."""
import numpy as np
import pytest
import torch   # here, not in a test: before any module's test loads the library, which then shares torch's HIP runtime

from kv4_near import PORTIONS, STEP, TOKENS, Held, attend, inputs, queries, why_not

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


class Cache:
    """sequences of given lengths as kv4_near.inputs makes them, in pages scattered over a pool whose bytes are 0xFF where no token is (codes 15, levels NaN)"""

    def __init__(self, lens, kv, hd, dtype, seed=0, scale=1.0):
        from tinygpt_amd import ops
        self.ops, self.lens, self.kv, self.hd, self.dtype = ops, lens, kv, hd, dtype
        self.first = np.concatenate([[0], np.cumsum(lens)])
        self.kx, self.vx = inputs(lens, kv, hd, dtype, seed, scale)
        need = [-(-n // 128) for n in lens]
        pages = sum(need) + 3
        order = np.random.default_rng(seed).permutation(pages)
        table = np.full((len(lens), max(need) + 1), -1, np.int32)
        for i, n in enumerate(need):
            table[i, :n], order = order[:n], order[n:]
        self.cache = ops.Kv4Cache(torch.full((1, pages, kv, hd * 144), 0xFF, dtype=torch.uint8, device="cuda"), torch.from_numpy(table).cuda(), kv, hd)
        self.k, self.v = (torch.from_numpy(x).to(DTYPES[dtype]).cuda() for x in (self.kx, self.vx))

    def part(self, parts):
        """(k, v, start, offsets) of [(sequence, from, to)]"""
        rows = np.concatenate([np.arange(self.first[i] + a, self.first[i] + b) for i, a, b in parts])
        at = torch.from_numpy(rows).cuda()
        return self.k[at], self.v[at], ints(a for _, a, _ in parts), ints(np.cumsum([0] + [b - a for _, a, b in parts]))

    def fill(self, upto=None):
        parts = [(i, 0, n) for i, n in enumerate(upto or self.lens) if n]
        if parts:
            k, v, start, off = self.part(parts)
            self.ops.kv4_append(self.cache, k, v, start, seq=ints(i for i, _, _ in parts), offsets=off)
        return self

    def held(self, i):
        s = slice(self.first[i], self.first[i + 1])
        return Held(self.kx[s]), Held(self.vx[s])

    def near(self, out, q, parts, window=0, scale=None, seen=None):
        """out, q [tokens of the parts][heads][hd]"""
        out, q, at = out.detach().double().cpu().numpy(), q.detach().double().cpu().numpy(), 0
        for i, a, b in parts:
            s = slice(at, at + b - a)
            at += b - a
            k, v = self.held(i)
            want, size = attend(q[s], k, v, list(range(a, b)), window, scale, seen)
            wrong = why_not(out[s], want, size, min(b, window or b), self.dtype)
            assert wrong is None, (i, a, b, wrong)


def on_gpu(x, dtype):
    return torch.from_numpy(x).to(DTYPES[dtype]).cuda()


# ---- every form, types and lengths -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens,group,kv", TOKENS)
def test_single_tokens(lens, group, kv, hd, dtype, fresh):
    parts = [(i, n - 1, n) for i, n in enumerate(lens)]
    c = Cache(lens, kv, hd, dtype, len(lens) + hd).fill([n - 1 for n in lens] if fresh else None)
    q = on_gpu(queries(len(lens), kv * group, hd, dtype, 9, 1.5), dtype)
    k, v, start, _ = c.part(parts)
    c.near(c.ops.kv4_attend(c.cache, q, start, max(lens), **(dict(k=k, v=v) if fresh else {})), q, parts)


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens,counts,group", PORTIONS)
def test_portions(lens, counts, group, hd, dtype, fresh):
    parts = [(i, n - c, n) for i, (n, c) in enumerate(zip(lens, counts))]
    c = Cache(lens, 2, hd, dtype, sum(lens)).fill([a for _, a, _ in parts] if fresh else None)
    k, v, start, off = c.part(parts)
    q = on_gpu(queries(len(k), 2 * group, hd, dtype, 8, 1.5), dtype)
    c.near(c.ops.kv4_attend(c.cache, q, start, max(lens), offsets=off, max_count=max(counts), **(dict(k=k, v=v) if fresh else {})), q, parts)


@pytest.mark.parametrize("window", [1, 2, 31, 100, 128, 129, 400, 5000])
@pytest.mark.parametrize("count,dtype", [(1, "fp16"), (1, "fp32"), (6, "bf16"), (6, "fp32"), (70, "fp16"), (70, "fp32")])
def test_windows(window, count, dtype):
    lens = [450, 128, 77]
    parts = [(i, max(0, n - count), n) for i, n in enumerate(lens)]
    c = Cache(lens, 2, 64, dtype, window).fill()
    _, _, start, off = c.part(parts)
    q = on_gpu(queries(sum(b - a for _, a, b in parts), 8, 64, dtype, 7), dtype)
    for i, n in enumerate(lens):
        c.cache.table[i, :max(0, n - count - window + 1) // 128] = -1      # pages that the window has left are gone
    c.near(c.ops.kv4_attend(c.cache, q, start, max(lens), offsets=off, window=window, max_count=count), q, parts, window)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("scale", [None, 1.0, -0.3, 0.0, 1e-6])
def test_scales_and_loud_scores(scale, dtype):
    c = Cache([600], 2, 64, dtype, 3, 4.0).fill()
    q = on_gpu(queries(1, 8, 64, dtype, 3, 30), dtype)
    c.near(c.ops.kv4_attend(c.cache, q, ints([599]), 600, scale=scale), q, [(0, 599, 600)], scale=scale)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("keys", [0, 1, 500, 3000, 200000])
def test_however_the_keys_are_divided(keys, dtype):
    c = Cache([3000], 2, 64, dtype, 1).fill()
    for count, group in [(1, 4), (3, 12), (20, 4)]:      # a lane a token; four waves that divide the keys; that divide the columns
        q = on_gpu(queries(count, 2 * group, 64, dtype, count), dtype)
        c.near(c.ops.kv4_attend(c.cache, q, ints([3000 - count]), keys, offsets=ints([0, count]), max_count=count), q, [(0, 3000 - count, 3000)])


@pytest.mark.parametrize("window", [0, 150])
@pytest.mark.parametrize("hd,group,gone,dtype", [(64, 4, [0], "fp32"), (128, 4, [1, 2], "bf16"), (64, 1, [3], "fp16"), (128, 7, [0, 2, 3], "fp32"), (64, 16, [0, 1, 2, 3], "fp32"), (128, 16, [0, 2], "fp16")])
def test_pages_that_are_not_there(hd, group, gone, dtype, window):
    n = 430
    c = Cache([n], 2, hd, dtype, hd + group).fill()
    c.cache.table[0, gone] = -1
    there = ~np.isin(np.arange(n) // 128, gone)
    for a in (0, 425, 429):      # a portion, a few tokens, one
        q = on_gpu(queries(n - a, 2 * group, hd, dtype, 4), dtype)
        out = c.ops.kv4_attend(c.cache, q, ints([a]), n, offsets=ints([0, n - a]), max_count=n - a, window=window)
        pick = sorted({a, n - 1} | {p for p in (0, 1, 31, 32, 127, 128, 200, 255, 256, 300, 383, 384) if p >= a})
        for p in pick:
            c.near(out[p - a:p - a + 1], q[p - a:p - a + 1], [(0, p, p + 1)], window, seen=there)


def test_32_bit_outputs_have_three_terms():
    """20 steps of 2^-24 over all heads of a row: 32-bit sums are within 10, and two 16-bit terms of a query or of a weight come to 38 and more (test_kv4_near.py)"""
    for n, hd in [(700, 64), (4096, 128)]:
        c = Cache([n], 1, hd, "fp32", n).fill()
        x = queries(1, 32, hd, "fp32", 5)
        want, _ = attend(x, *c.held(0), [n - 1])
        for group in (8, 16):      # single tokens' kernel; four waves that divide the keys
            out = torch.cat([c.ops.kv4_attend(c.cache, on_gpu(x[:, h:h + group].copy(), "fp32"), ints([n - 1]), n) for h in range(0, 32, group)], 1)
            off = np.sqrt(((out.double().cpu().numpy() - want) ** 2).sum() / (want ** 2).sum())
            assert off < 20 * 2.0 ** -24, (n, hd, group, off)


# ---- long walks ------------------------------------------------------------------------------------------------------------------------------------------
def long_rows(n, count, group, kv, hd, dtype, rows=1, pick=6):
    """(mean square of the error, of the right values' rounding, of the right values) over some tokens of `rows` entries that bring `count` tokens each to one sequence of n"""
    from tinygpt_amd import ops
    g = torch.Generator("cuda").manual_seed(n + count + hd)
    t = DTYPES[dtype]
    pages = -(-n // 128)
    cache = ops.Kv4Cache.empty(1, pages, kv, hd, rows, n)
    cache.table[:] = torch.randperm(pages, device="cuda", generator=g).int()[None]
    k = (torch.randn(n, kv, hd, device="cuda", generator=g) + 0.7 * torch.randn(kv, hd, device="cuda", generator=g)).to(t)
    v = torch.randn(n, kv, hd, device="cuda", generator=g).to(t)
    whole = dict(seq=ints([0]), offsets=ints([0, n]))
    ops.kv4_append(cache, k, v, ints([0]), **whole)
    k, v = (x.double() for x in ops.kv4_read(cache, ints([0]), n, **whole))
    q = torch.randn(rows * count, kv * group, hd, device="cuda", generator=g).to(t)
    out = ops.kv4_attend(cache, q, ints([n - count] * rows), n, offsets=ints(range(0, rows * count + 1, count)) if count > 1 else None, max_count=count)
    sums = torch.zeros(3, dtype=torch.float64, device="cuda")
    for i in sorted({int(x) for x in np.linspace(0, rows * count - 1, pick)}):
        p = n - count + i % count + 1
        for h in range(kv):
            hs = slice(h * group, h * group + group)
            w = torch.softmax(q[i, hs].double() @ k[:p, h].T.contiguous() / hd ** 0.5, -1)
            want = w @ v[:p, h]
            sums += torch.stack([((out[i, hs].double() - want) ** 2).sum(), ((want.to(t).double() - want) ** 2).sum(), (want ** 2).sum()])
    return sums.tolist()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n,count,group,kv,hd,rows", [(32768, 1024, 16, 2, 128, 1), (32768, 1024, 16, 2, 64, 1), (131072, 1, 4, 8, 128, 64), (131072, 1, 8, 8, 64, 64), (131072, 1, 16, 8, 64, 64), (131072, 5, 4, 8, 128, 48),
                                                      (131072, 2, 4, 8, 64, 64)])
def test_long_walks_leave_an_output_its_rounding(n, count, group, kv, hd, rows, dtype):
    """Keys that one workgroup walks from the first to the last, outputs in 16 bits: the error beside the rounding of the output is 2^-14 of a row's rms at most (kv4_near.own), however long the
    walk.  Sums that take the codes of all keys before the los join them are off by 2^-24 of themselves a product, 4e-4 of the row at 32768 keys."""
    err, rounding, size = long_rows(n, count, group, kv, hd, dtype, rows)
    assert err <= 1.02 * rounding + (2.0 ** -14) ** 2 * size, ((err / size) ** 0.5, (rounding / size) ** 0.5)
    assert rounding <= STEP[dtype] ** 2 / 3 * size
