"""Operators on a 4-bit cache (tinygpt_amd.ops, kernels/kv4.h) against their definitions in 64 bits (kv4_util.py), bit for bit where the definition says which bits."""
import numpy as np
import pytest
import torch as _torch   # here, not in a test: before any module's test loads the library, which then shares torch's HIP runtime

from kv4_util import PAGE, attend, bound, quantise, values

pytestmark = pytest.mark.gpu

EPS = {"bf16": 2.0 ** -7, "fp16": 2.0 ** -10, "fp32": 2.0 ** -23}


@pytest.fixture(scope="module")
def torch():
    return _torch


def dtype_of(torch, name):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[name]


def numpy_of(t):
    return t.detach().float().cpu().numpy()


def ints(torch, x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


class Rows:
    """Sequences of given lengths in a cache whose pages lie scattered over a pool, everything that no token fills set to 0xFF bytes (codes 15, levels NaN)"""

    def __init__(self, torch, lens, kv_heads, hd, dtype, seed=0, spare=3, layers=1, layer=0, room=0, scale=1.0):
        from tinygpt_amd import ops
        self.torch, self.ops, self.lens, self.layer = torch, ops, list(lens), layer
        rng = np.random.default_rng(seed)
        need = [-(-(n + room) // PAGE) for n in lens]
        pages = sum(need) + spare
        order = rng.permutation(pages)
        table = np.full((len(lens), max(need + [1]) + 1), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        self.unused = order[at:]
        self.cache = ops.Kv4Cache(torch.full((layers, pages, kv_heads, hd * 144), 0xFF, dtype=torch.uint8, device="cuda"), torch.from_numpy(table).cuda(), kv_heads, hd)
        off = rng.normal(size=(kv_heads, hd)) * 0.7
        total = sum(lens) + room * len(lens)
        t = dtype_of(torch, dtype)
        self.k = torch.tensor(scale * (rng.normal(size=(total, kv_heads, hd)) + off), dtype=torch.float32).to(t).cuda()
        self.v = torch.tensor(scale * rng.normal(size=(total, kv_heads, hd)), dtype=torch.float32).to(t).cuda()
        self.first = np.concatenate([[0], np.cumsum(np.array(lens, np.int64) + room)])

    def span(self, i, a, b):
        return slice(int(self.first[i] + a), int(self.first[i] + b))

    def rows(self, parts):
        """(k, v, start, offsets) of parts [(sequence, from, to)] as one batch"""
        torch = self.torch
        k = torch.cat([self.k[self.span(*p)] for p in parts])
        v = torch.cat([self.v[self.span(*p)] for p in parts])
        return k, v, ints(torch, [p[1] for p in parts]), ints(torch, np.concatenate([[0], np.cumsum([p[2] - p[1] for p in parts])]))

    def fill(self, upto=None):
        parts = [(i, 0, n if upto is None else upto[i]) for i, n in enumerate(self.lens)]
        parts = [p for p in parts if p[2] > 0]
        if parts:
            k, v, start, off = self.rows(parts)
            self.ops.kv4_append(self.cache, k, v, start, self.layer, seq=ints(self.torch, [p[0] for p in parts]), offsets=off)
        return self

    def held(self, i):
        s = self.span(i, 0, self.lens[i])
        return values(numpy_of(self.k[s])), values(numpy_of(self.v[s]))


def check(out, rows, seqs, pos, q, dtype, window=0, scale=None):
    """out, q [T][heads][hd]: token t of sequence seqs[t] at pos[t]"""
    out, q = numpy_of(out).astype(np.float64), numpy_of(q).astype(np.float64)
    for i in sorted(set(seqs)):
        mine = [t for t, s in enumerate(seqs) if s == i]
        (k, kb), (v, vb) = rows.held(i)
        want, s, o = attend(q[mine], k, v, [pos[t] for t in mine], window, scale, (kb, vb))
        b = bound(want, s, o, len(k), EPS[dtype], 1 if dtype == "bf16" else 2)
        bad = np.abs(out[mine] - want) > b
        assert not bad.any(), (i, float((np.abs(out[mine] - want) / b).max()), [int(x) for x in np.argwhere(bad)[0]])


# ---- append and read ---------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hd", [64, 128])
def test_append_keeps_exactly_the_levels_of_the_format(torch, hd, dtype):
    """portions that begin and end inside words, blocks and pages, then single tokens; read back as float32: bit for bit"""
    r = Rows(torch, [1, 31, 32, 129, 200, 517], 3, hd, dtype, seed=hd)
    cuts = [(1,), (7, 31), (3, 5, 32), (128, 129), (1, 2, 3, 4, 33, 95, 127, 200), (5, 261, 517)]
    done = [0] * 6
    for step in range(8):
        parts = []
        for i, c in enumerate(cuts):
            if step < len(c):
                parts.append((i, done[i], c[step]))
                done[i] = c[step]
        if parts:
            k, v, start, off = r.rows(parts)
            r.ops.kv4_append(r.cache, k, v, start, seq=ints(torch, [p[0] for p in parts]), offsets=off)
    assert done == r.lens
    k, v, start, off = r.rows([(i, 0, n) for i, n in enumerate(r.lens)])
    ko, vo = r.ops.kv4_read(r.cache, start, len(k), offsets=off)
    for got, src in ((ko, k), (vo, v)):
        n, lo, step = quantise(numpy_of(src))
        want = (np.repeat(lo.astype(np.float64), 64, -1) + np.repeat(step.astype(np.float64), 64, -1) * n).astype(np.float32)
        assert np.array_equal(numpy_of(got), want)
    # the same tokens one at a time give the same bytes
    one = Rows(torch, r.lens, 3, hd, dtype, seed=hd)
    for t in range(max(r.lens)):
        parts = [(i, t, t + 1) for i, n in enumerate(r.lens) if t < n]
        k, v, start, off = one.rows(parts)
        one.ops.kv4_append(one.cache, k, v, start, seq=ints(torch, [p[0] for p in parts]))
    assert torch.equal(one.cache.pool, r.cache.pool)


def test_append_of_levels_at_their_edges(torch):
    """constant groups, zeros of both signs, one loud channel, numbers of 1e30 and 1e-30, ties between levels, values that are not finite"""
    r = Rows(torch, [40], 1, 128, "fp32")
    x = np.random.default_rng(5).normal(size=(40, 1, 128)).astype(np.float32)
    x[0] = 0; x[1] = -0.0; x[2] = 3.7; x[3] *= 1e30; x[4] *= 1e-30; x[5, 0, 9] = 1e6
    x[6] = np.tile(np.arange(64) % 16, 2)                        # lo 0, step 1: exactly the levels
    x[7] = np.tile((np.arange(64) % 31) / 2, 2)                  # ties
    x[8, 0, 3] = np.inf; x[9, 0, 70] = -np.inf; x[10, 0, 0] = np.nan; x[11] = 3.4e38; x[11, 0, 0] = -3.4e38; x[12] = 1e-44
    r.k = torch.from_numpy(x).cuda(); r.v = torch.from_numpy(x[::-1].copy()).cuda()
    for way in ("portion", "tokens"):
        r.cache.pool.fill_(0xFF)
        if way == "portion":
            r.fill()
        else:
            for t in range(40):
                r.ops.kv4_append(r.cache, r.k[t:t + 1], r.v[t:t + 1], ints(torch, [t]))
        ko, vo = r.ops.kv4_read(r.cache, ints(torch, [0]), 40, offsets=ints(torch, [0, 40]))
        for got, src in ((ko, x), (vo, x[::-1])):
            n, lo, step = quantise(src)
            want = (np.repeat(lo.astype(np.float64), 64, -1) + np.repeat(step.astype(np.float64), 64, -1) * n).astype(np.float32)
            assert np.array_equal(numpy_of(got), want, equal_nan=True), way
        assert np.isnan(numpy_of(ko)[8, 0, :64]).all() and not np.isnan(numpy_of(ko)[8, 0, 64:]).any() and np.isnan(numpy_of(ko)[9, 0, 64:]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_read_rounds_once(torch, dtype):
    r = Rows(torch, [300], 2, 64, dtype).fill()
    k, v = r.ops.kv4_read(r.cache, ints(torch, [0]), 300, dtype=dtype_of(torch, dtype), offsets=ints(torch, [0, 300]))
    k32, v32 = r.ops.kv4_read(r.cache, ints(torch, [0]), 300, offsets=ints(torch, [0, 300]))
    assert torch.equal(k, k32.to(k.dtype)) and torch.equal(v, v32.to(v.dtype))
    s = values(numpy_of(r.k))[0]
    assert np.array_equal(numpy_of(k32), s.astype(np.float32))


def test_append_leaves_the_rest_of_the_pool(torch):
    """pages of others, tokens of the same words, other layers; tokens without a page, before position 0, behind the table or of sequences that are not there"""
    r = Rows(torch, [200, 90], 2, 64, "bf16", layers=3, layer=1).fill()
    before = r.cache.pool.clone()
    k, v, start, off = r.rows([(0, 5, 6)])
    r.ops.kv4_append(r.cache, k, v, ints(torch, [5]), 1, seq=ints(torch, [0]))      # what is there already
    assert torch.equal(before, r.cache.pool)
    T = r.cache.table.shape[1] * PAGE
    for start, seq in [(T, 0), (T + 7, 0), (2 ** 31 - 1, 0), (-1, 0), (-2 ** 31, 0), (130, 1), (5, 2), (5, -1), (5, 2 ** 31 - 1)]:
        r.ops.kv4_append(r.cache, k, v, ints(torch, [start]), 1, seq=ints(torch, [seq]))
        assert torch.equal(before, r.cache.pool), (start, seq)
    k, v, start, off = r.rows([(0, 0, 40)])
    for offs in [(0, 41), (-1, 40), (30, 20), (2 ** 31 - 1, 2 ** 31 - 1)]:
        r.ops.kv4_append(r.cache, k, v, ints(torch, [300]), 1, offsets=ints(torch, offs), max_count=40)
        assert torch.equal(before, r.cache.pool), offs
    for bad in (-5, r.cache.pool.shape[1], 2 ** 31 - 1):
        r.cache.table[1, 0] = bad
        r.ops.kv4_append(r.cache, k, v, ints(torch, [3]), 1, seq=ints(torch, [1]), offsets=ints(torch, [0, 40]))
        r.ops.kv4_append(r.cache, k[:1], v[:1], ints(torch, [3]), 1, seq=ints(torch, [1]))
        assert torch.equal(before, r.cache.pool), bad
        ko, vo = r.ops.kv4_read(r.cache, ints(torch, [3]), 40, layer=1, seq=ints(torch, [1]), offsets=ints(torch, [0, 40]))
        assert not ko.any() and not vo.any()
    with pytest.raises(ValueError):
        r.ops.kv4_append(r.cache, k[:1], v[:1], ints(torch, [3]), 3)
    # tokens that straddle a position 0: those from it on
    r2 = Rows(torch, [30], 1, 64, "bf16", seed=3)
    kk, vv = r2.k[:30], r2.v[:30]
    r2.ops.kv4_append(r2.cache, kk, vv, ints(torch, [-10]), offsets=ints(torch, [0, 30]))
    ko, _ = r2.ops.kv4_read(r2.cache, ints(torch, [0]), 20, offsets=ints(torch, [0, 20]))
    assert np.array_equal(numpy_of(ko), values(numpy_of(kk[10:]))[0].astype(np.float32))


# ---- attention ---------------------------------------------------------------------------------------------------------------------------------------------
TOKENS = [([1], 4, 1), ([2, 1, 33], 4, 1), ([127, 128, 129, 130], 1, 1), ([713], 4, 1), ([300, 5, 1000], 7, 1), ([64, 700], 16, 1), ([257, 31], 2, 1)]


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens,group,kv_heads", TOKENS + [([513, 90], 3, 5)])
def test_single_tokens(torch, lens, group, kv_heads, hd, dtype, fresh):
    r = Rows(torch, lens, kv_heads, hd, dtype, seed=len(lens) + hd)
    r.fill([n - 1 for n in lens] if fresh else None)
    q = torch.tensor(np.random.default_rng(9).normal(size=(len(lens), kv_heads * group, hd)) * 1.5, dtype=torch.float32).to(dtype_of(torch, dtype)).cuda()
    k, v, start, _ = r.rows([(i, n - 1, n) for i, n in enumerate(lens)])
    new = dict(k=k, v=v) if fresh else {}
    out = r.ops.kv4_attend(r.cache, q, start, max(lens), **new)
    check(out, r, list(range(len(lens))), [n - 1 for n in lens], q, dtype)
    if fresh:      # the same bits as an append and a call without it, and what was appended is what an append gives
        two = Rows(torch, lens, kv_heads, hd, dtype, seed=len(lens) + hd).fill()
        assert torch.equal(two.cache.pool, r.cache.pool)
        assert torch.equal(out, r.ops.kv4_attend(r.cache, q, start, max(lens)))


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("hd,dtype", [(64, "bf16"), (128, "bf16"), (64, "fp16"), (128, "fp32")])
@pytest.mark.parametrize("lens,counts,group", [([5], [5], 4), ([40, 3, 260], [2, 3, 5], 4), ([130, 700], [9, 8], 1), ([300], [300], 1), ([290, 33, 129], [70, 33, 1], 4), ([1000], [150], 7), ([200, 64], [17, 30], 16)])
def test_portions(torch, lens, counts, group, hd, dtype, fresh):
    r = Rows(torch, lens, 2, hd, dtype, seed=sum(lens))
    parts = [(i, n - c, n) for i, (n, c) in enumerate(zip(lens, counts))]
    r.fill([p[1] for p in parts] if fresh else None)
    k, v, start, off = r.rows(parts)
    q = torch.tensor(np.random.default_rng(8).normal(size=(len(k), 2 * group, hd)), dtype=torch.float32).to(dtype_of(torch, dtype)).cuda()
    out = r.ops.kv4_attend(r.cache, q, start, max(lens), offsets=off, max_count=max(counts), **(dict(k=k, v=v) if fresh else {}))
    check(out, r, [p[0] for p in parts for _ in range(p[2] - p[1])], [t for p in parts for t in range(p[1], p[2])], q, dtype)


@pytest.mark.parametrize("window", [1, 2, 31, 100, 128, 129, 400, 5000])
@pytest.mark.parametrize("count", [1, 6, 70])
def test_windows(torch, window, count):
    lens = [450, 128, 77]
    r = Rows(torch, lens, 2, 64, "fp16", seed=window).fill()
    parts = [(i, max(0, n - count), n) for i, n in enumerate(lens)]
    _, _, start, off = r.rows(parts)
    T = sum(p[2] - p[1] for p in parts)
    q = torch.tensor(np.random.default_rng(7).normal(size=(T, 8, 64)), dtype=torch.float32).half().cuda()
    # pages that the window has left hold anything, or are gone
    for i, n in enumerate(lens):
        gone = max(0, n - count - window + 1) // PAGE
        r.cache.table[i, :gone] = -1
    out = r.ops.kv4_attend(r.cache, q, start, max(lens), offsets=off, window=window, max_count=count)
    check(out, r, [p[0] for p in parts for _ in range(p[2] - p[1])], [t for p in parts for t in range(p[1], p[2])], q, "fp16", window)


def test_scale_and_loud_scores(torch):
    """scores of thousands, a scale of its own, negative and zero"""
    r = Rows(torch, [600], 2, 64, "fp32", scale=4.0).fill()
    q = torch.tensor(np.random.default_rng(3).normal(size=(1, 8, 64)) * 30, dtype=torch.float32).cuda()
    for scale in (None, 1.0, -0.3, 0.0, 1e-6):
        out = r.ops.kv4_attend(r.cache, q, ints(torch, [599]), 600, scale=scale)
        check(out, r, [0], [599], q, "fp32", scale=scale)


def test_rows_that_see_nothing_are_zero_and_others_stay(torch):
    r = Rows(torch, [300, 40], 2, 64, "bf16").fill()
    q = torch.randn(6, 8, 64, device="cuda").bfloat16()
    # entries: before position 0; a sequence that is not there; a good one; nothing at all
    out = torch.full_like(q, 7.0)
    r.ops.kv4_attend(r.cache, q, ints(torch, [-1, 5, 39, 3]), 300, seq=ints(torch, [0, 9, 1, 0]), offsets=ints(torch, [0, 1, 2, 4, 4]), out=out)
    assert not out[0].any() and (out[1] == 7).all() and (out[4:] == 7).all()
    check(out[2:3], r, [1], [39], q[2:3], "bf16")
    # every page gone: zeros, whatever the division of the keys
    r.cache.table.fill_(-1)
    for keys in (300, 100000):
        assert not r.ops.kv4_attend(r.cache, q[:2], ints(torch, [299, 39]), keys).any()
        assert not r.ops.kv4_attend(r.cache, q, ints(torch, [290]), keys, offsets=ints(torch, [0, 6])).any()


def test_pages_that_are_not_there_are_not_seen(torch):
    r = Rows(torch, [400], 2, 128, "fp32").fill()
    q = torch.randn(1, 8, 128, device="cuda")
    good = r.cache.table.clone()
    for bad in (-1, r.cache.pool.shape[1], 2 ** 31 - 1, -2 ** 31):
        r.cache.table.copy_(good)
        r.cache.table[0, 1] = bad
        out = numpy_of(r.ops.kv4_attend(r.cache, q, ints(torch, [399]), 400)).astype(np.float64)
        (k, kb), (v, vb) = r.held(0)
        keep = np.r_[0:128, 256:400]
        want, s, o = attend(numpy_of(q), k[keep], v[keep], [len(keep) - 1], big=(kb[keep], vb[keep]))
        assert (np.abs(out - want) <= bound(want, s, o, 400, EPS["fp32"], 2)).all()


@pytest.mark.parametrize("window", [0, 150])
@pytest.mark.parametrize("hd,group,gone", [(64, 4, [0]), (128, 4, [1, 2]), (64, 1, [3]), (128, 7, [0, 2, 3]), (64, 16, [0, 1, 2, 3])])
def test_portions_over_pages_that_are_not_there(torch, hd, group, gone, window):
    """tokens -7 .. 429 of a sequence some of whose pages are missing, several workgroups of columns"""
    n, before = 430, 7
    r = Rows(torch, [n], 2, hd, "fp32", seed=hd + group).fill()
    r.cache.table[0, gone] = -1
    q = torch.tensor(np.random.default_rng(4).normal(size=(n + before, 2 * group, hd)), dtype=torch.float32).cuda()
    out = numpy_of(r.ops.kv4_attend(r.cache, q, ints(torch, [-before]), n, offsets=ints(torch, [0, n + before]), window=window)).astype(np.float64)
    (k, kb), (v, vb) = r.held(0)
    there = np.array([p for p in range(n) if p // PAGE not in gone], int)
    for t in list(range(before)) + [before + p for p in (0, 1, 31, 32, 127, 128, 200, 255, 256, 300, 383, 384, 429)]:
        pos = t - before
        keep = there[(there <= pos) & ((window == 0) | (there > pos - window))]
        if not len(keep):
            assert not out[t].any()
            continue
        want, s, o = attend(numpy_of(q[t:t + 1]), k[keep], v[keep], [len(keep) - 1], big=(kb[keep], vb[keep]))
        assert (np.abs(out[t:t + 1] - want) <= bound(want, s, o, n, EPS["fp32"], 2)).all(), t


def test_positions_behind_the_table_see_its_pages(torch):
    r = Rows(torch, [256], 1, 64, "bf16").fill()
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()
    out = r.ops.kv4_attend(r.cache, q, ints(torch, [2 ** 31 - 2]), 2 ** 31 - 1)
    check(out, r, [0], [2 ** 31 - 2], q, "bf16")


def test_max_keys_and_division_do_not_change_what_is_seen(torch):
    r = Rows(torch, [3000], 2, 64, "fp32").fill()
    q = torch.randn(1, 8, 64, device="cuda")
    for keys in (0, 1, 500, 3000, 200000):
        check(r.ops.kv4_attend(r.cache, q, ints(torch, [2999]), keys), r, [0], [2999], q, "fp32")


def test_values_that_are_not_finite(torch):
    """a group with one reads as NaN where it is seen, and is nothing where it is not"""
    r = Rows(torch, [150], 1, 128, "fp32")
    r.v[100, 0, 3] = np.inf
    r.fill()
    q = torch.randn(2, 4, 128, device="cuda")
    out = r.ops.kv4_attend(r.cache, q, ints(torch, [98]), 150, offsets=ints(torch, [0, 2]))
    check(out, r, [0, 0], [98, 99], q, "fp32")
    out = numpy_of(r.ops.kv4_attend(r.cache, q, ints(torch, [99]), 150, offsets=ints(torch, [0, 2])))
    assert np.isfinite(out[0]).all() and np.isnan(out[1, :, :64]).all() and np.isfinite(out[1, :, 64:]).all()
    out = numpy_of(r.ops.kv4_attend(r.cache, q[:1], ints(torch, [149]), 150, window=49))
    assert np.isfinite(out).all()
    r.k[120, 0, 0] = np.nan
    r.fill()
    assert np.isnan(numpy_of(r.ops.kv4_attend(r.cache, q[:1], ints(torch, [149]), 150))).all()


def test_strides(torch):
    """queries, keys, values and outputs as parts of a larger product's rows, heads first, at odd offsets; the table as a part of a larger one"""
    kv, hd, group, lens = 2, 64, 4, [130, 61, 300]
    r = Rows(torch, lens, kv, hd, "bf16")
    wide = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    wide[:, 5:5 + r.cache.table.shape[1]] = r.cache.table
    r.cache = r.ops.Kv4Cache(r.cache.pool, wide[:, 5:5 + r.cache.table.shape[1]], kv, hd)
    for odd in (0, 1, 3):
        for heads_first in (False, True):
            for count in (1, 33):
                parts = [(i, n - count, n) for i, n in enumerate(lens)]
                r.fill([p[1] for p in parts])
                k, v, start, off = r.rows(parts)
                T = len(k)
                q = torch.randn(T, kv * group, hd, device="cuda").bfloat16()
                flat = torch.zeros(T * ((group + 2) * kv * hd + 7) + odd, dtype=torch.bfloat16, device="cuda")[odd:]
                if heads_first:
                    rows = flat[:T * (group + 2) * kv * hd].view((group + 2) * kv, T, hd).transpose(0, 1)
                else:
                    rows = flat.view(T, -1)[:, :(group + 2) * kv * hd].unflatten(1, (-1, hd))
                rows[:, :kv * group] = q; rows[:, kv * group:kv * group + kv] = k; rows[:, kv * group + kv:] = v
                out = torch.zeros(kv * group, T + 1, hd + odd, dtype=torch.bfloat16, device="cuda")
                o = r.ops.kv4_attend(r.cache, rows[:, :kv * group], start, max(lens), offsets=off, max_count=count, k=rows[:, kv * group:kv * group + kv], v=rows[:, kv * group + kv:],
                                     out=out[:, :T, odd:].transpose(0, 1))
                check(o, r, [p[0] for p in parts for _ in range(count)], [t for p in parts for t in range(p[1], p[2])], q, "bf16")
                assert not out[:, T].any() and not out[..., :odd].any()


def test_offsets_beyond_32_bits(torch):
    """pages whose places in the pool pass 2^32 bytes and words"""
    from tinygpt_amd import ops
    kv, hd, pages = 8, 128, 130000      # 19 GB
    pool = torch.empty(1, pages, kv * hd * 144, dtype=torch.uint8, device="cuda")
    table = ints(torch, [pages - 1, 3, 129999 - 15000, 60000, 0, 33000]).view(1, -1)
    r = Rows(torch, [700], kv, hd, "bf16")
    r.cache = ops.Kv4Cache(pool, table, kv, hd)
    r.fill([699])
    q = torch.randn(1, 32, hd, device="cuda").bfloat16()
    out = ops.kv4_attend(r.cache, q, ints(torch, [699]), 700, k=r.k[699:700], v=r.v[699:700])
    check(out, r, [0], [699], q, "bf16")
    ops.copy_pages(pool, ints(torch, [pages - 1, 60000]), ints(torch, [pages - 7, 59000]))
    table[0, 0] = pages - 7; table[0, 3] = 59000
    assert torch.equal(out, ops.kv4_attend(r.cache, q, ints(torch, [699]), 700))


# ---- pages -----------------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layers,pages,shape,dtype", [(1, 5, (4,), "int32"), (3, 9, (8, 128, 64), "int16"), (2, 40, (2, 64 * 144), "uint8"), (4, 7, (40000,), "int32"), (2, 3, (1, 1, 8), "int16")])
def test_copied_pages(torch, layers, pages, shape, dtype):
    from tinygpt_amd import ops
    g = torch.Generator("cuda").manual_seed(1)
    pool = torch.randint(0, 120, (layers, pages, *shape), generator=g, device="cuda").to(getattr(torch, dtype))
    at = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    n = pages // 2
    want = pool.clone()
    want[:, at[n:2 * n].long()] = pool[:, at[:n].long()]
    other = torch.zeros(layers, pages + 3, *shape, dtype=pool.dtype, device="cuda")
    ops.copy_pages(pool, at[:n], at[n:2 * n], into=other)
    assert torch.equal(other[:, at[n:2 * n].long()], pool[:, at[:n].long()]) and int((other != 0).flatten(2).any(2).sum()) <= layers * n
    ops.copy_pages(pool, at[:n], at[n:2 * n])
    assert torch.equal(pool, want)
    # pairs with a page that is not there, and none at all
    ops.copy_pages(pool, ints(torch, [-1, pages, 0, 0, 2 ** 31 - 1]), ints(torch, [0, 0, pages, -1, 1]))
    ops.copy_pages(pool, at[:0], at[:0])
    assert torch.equal(pool, want)


# ---- as they are used ----------------------------------------------------------------------------------------------------------------------------------------
def test_prompt_tokens_fork_and_compaction(torch):
    """a prompt in portions, tokens one by one, a fork that shares whole pages and copies the last, both rows going on, a smaller pool: outputs all along"""
    from tinygpt_amd import ops
    kv, hd, group, layers = 2, 64, 4, 3
    r = Rows(torch, [300, 300], kv, hd, "bf16", layers=layers, room=0, spare=6)
    r.k[300:450], r.v[300:450] = r.k[:150].clone(), r.v[:150].clone()      # the fork: the same first 150 tokens
    table = r.cache.table
    pages = r.cache.pool.shape[1]
    table.fill_(-1)
    table[0, :3] = ints(torch, [4, 0, 7])
    g = torch.Generator("cuda").manual_seed(4)

    def step(seqs, starts, count):
        q = torch.randn(len(seqs) * count, kv * group, hd, generator=g, device="cuda").bfloat16()
        parts = [(s, a, a + count) for s, a in zip(seqs, starts)]
        k, v, start, off = r.rows(parts)
        outs = [ops.kv4_attend(r.cache, q, start, 300, layer, seq=ints(torch, seqs), offsets=off if count > 1 else None, max_count=count, k=k, v=v) for layer in range(layers)]
        for o in outs[1:]:
            assert torch.equal(o, outs[0])
        check(outs[0], r, [p[0] for p in parts for _ in range(count)], [t for p in parts for t in range(p[1], p[2])], q, "bf16")

    step([0], [0], 64)
    step([0], [64], 83)
    for t in range(147, 150):
        step([0], [t], 1)
    table[1, 0] = table[0, 0]                                               # whole pages are shared, the one that goes on is copied
    table[1, 1] = 8
    ops.copy_pages(r.cache.pool, table[0, 1:2], table[1, 1:2].clone())
    table[1, 2] = 2
    for t in range(150, 160):
        step([1, 0], [t, t], 1)
    step([0, 1], [160, 160], 100)
    small = torch.zeros(layers, 5, *r.cache.pool.shape[2:], dtype=torch.uint8, device="cuda")      # the five pages in use, moved together
    used = ints(torch, sorted({int(x) for x in table.flatten() if x >= 0}))
    assert len(used) == 5 and pages > 5
    ops.copy_pages(r.cache.pool, used, ints(torch, range(5)), into=small)
    moved = torch.full_like(table, -1)
    for i, p in enumerate(used.tolist()):
        moved[table == p] = i
    r.cache.pool.fill_(0xFF)
    r.cache = ops.Kv4Cache(small, moved, kv, hd)
    for t in range(260, 300):
        step([0, 1], [t, t], 1)


def test_streams_and_graphs(torch):
    """another stream than the default; a captured step replayed while positions, queries and pages change, with other work between; two graphs with workspaces of their own"""
    from tinygpt_amd import ops
    r = Rows(torch, [700, 300], 2, 64, "bf16", room=0).fill([400, 100])
    side = torch.cuda.Stream()
    q = torch.randn(2, 8, 64, device="cuda").bfloat16()
    start = ints(torch, [400, 100])
    k, v = r.k[[400, 800]].clone(), r.v[[400, 800]].clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops.kv4_attend(r.cache, q, start, 700, k=k, v=v)
    torch.cuda.current_stream().wait_stream(side)
    check(out, r, [0, 1], [400, 100], q, "bf16")
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = ops.kv4_attend(r.cache, q, start, 700, k=k, v=v)
            kk, vv = ops.kv4_read(r.cache, start, 2)
        graphs.append((g, o, kk, vv))
    for t in range(1, 60):
        start.copy_(ints(torch, [400 + t, 100 + t]))
        q.normal_()
        k.copy_(r.k[[400 + t, 800 + t]]); v.copy_(r.v[[400 + t, 800 + t]])
        g, o, kk, vv = graphs[t % 2]
        g.replay()
        if t % 3 == 0:
            torch.cuda.synchronize()
        eager = ops.kv4_attend(r.cache, q, start, 700)
        assert torch.equal(o, eager), t
        assert torch.equal(kk, ops.kv4_read(r.cache, start, 2)[0])
        if t % 20 == 0:
            check(o, r, [0, 1], [400 + t, 100 + t], q, "bf16")
        torch.randn(1 << 20, device="cuda").sum()


@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("heads,n", [(2, 700), (8, 90), (32, 300)])
def test_entries_of_one_sequence_see_each_other(torch, heads, n, offsets):
    """the last tokens of a sequence as entries of one token each, in any order: as appended first, bit for bit"""
    new = 9
    rows = [Rows(torch, [n], 2, 64, "bf16", room=new).fill() for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(new, heads, 64, device="cuda", generator=g).bfloat16()
    order = [4, 8, 0, 7, 3, 1, 6, 2, 5]
    k = torch.stack([rows[0].k[n + i] for i in order])
    v = torch.stack([rows[0].v[n + i] for i in order])
    batch = dict(seq=ints(torch, [0] * new), offsets=ints(torch, range(new + 1)) if offsets else None, max_count=1 if offsets else None)
    start = ints(torch, [n + i for i in order])
    out = rows[0].ops.kv4_attend(rows[0].cache, q, start, n + new, k=k, v=v, **batch)
    rows[1].ops.kv4_append(rows[1].cache, k, v, start, **batch)
    want = rows[1].ops.kv4_attend(rows[1].cache, q, start, n + new, **batch)
    assert torch.equal(out, want) and torch.equal(rows[0].cache.pool, rows[1].cache.pool)


def test_same_call_same_bits(torch):
    r = Rows(torch, [5000, 60], 4, 128, "bf16").fill()
    q = torch.randn(2, 16, 128, device="cuda").bfloat16()
    a = r.ops.kv4_attend(r.cache, q, ints(torch, [4999, 59]), 5000)
    for _ in range(5):
        assert torch.equal(a, r.ops.kv4_attend(r.cache, q, ints(torch, [4999, 59]), 5000))


def test_refused_tensors(torch):
    r = Rows(torch, [10], 2, 64, "bf16").fill()
    ops, c = r.ops, r.cache
    q, s = torch.randn(1, 8, 64, device="cuda").bfloat16(), ints(torch, [9])
    for args, more in [((q[0], s, 10), {}), ((q.float().double(), s, 10), {}), ((q.cpu(), s, 10), {}), ((q, s.long(), 10), {}), ((q, s.cpu(), 10), {}), ((q, s, 10), dict(k=r.k[:1])),
                       ((q, s, 10), dict(k=r.k[:2], v=r.v[:2])), ((q.repeat(2, 1, 1), s, 10), {}), ((q, s, 10), dict(offsets=s)), ((q, s, 10), dict(out=q.float())), ((q, s, 10), dict(layer=1)),
                       ((torch.randn(1, 8, 128, device="cuda").bfloat16()[..., ::2], s, 10), {}), ((torch.randn(1, 8, 128, device="cuda").bfloat16(), s, 10), {})]:
        with pytest.raises(ValueError):
            ops.kv4_attend(c, *args, **more)
    from tinygpt_amd.ffi import TgxError
    for args, more in [((q[:, :7], s, 10), {}), ((q, s, 10), dict(window=-1)), ((q, s, -1), {}), ((q, s, 10), dict(scale=float("nan")))]:
        with pytest.raises(TgxError):
            ops.kv4_attend(c, *args, **more)
    assert ops.kv4_attend(c, q[:0], s[:0], 10).shape == (0, 8, 64)


def test_tensors_that_ask_for_gradients_are_refused(torch):
    r = Rows(torch, [5], 1, 64, "bf16", room=1).fill()
    start = ints(torch, [4])
    q = torch.zeros(1, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        r.ops.kv4_attend(r.cache, q, start, 5)
    with pytest.raises(ValueError, match="gradient"):
        r.ops.kv4_append(r.cache, r.k[5:].clone().requires_grad_(), r.v[5:], start)
    with torch.no_grad():
        assert not r.ops.kv4_attend(r.cache, q, start, 5).requires_grad
