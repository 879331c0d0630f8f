"""Calls of the 4-bit cache, its operators and the forks that one might not think of: what a refusal leaves, sizes of zero, large batches, pending tokens."""
import ctypes

import numpy as np
import pytest
import torch   # here, not in a test: before any module's test loads the library, which then shares torch's HIP runtime

from test_hip_kv4_model import ids, make
from tinygpt_amd.ffi import GREEDY, SamplerCfg, TgxError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from tinygpt_amd.ffi import product_backend
    return product_backend()


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


# ---- models ----------------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("missing", ["keys", "values"])
def test_a_refused_write_leaves_a_fork_its_shared_blocks(missing, hip):
    m, _ = make("llama_tiny", hip, "bf16", 4, max_batch=2, budget=1024)
    m.forward_row(0, ids(np.random.default_rng(1), 300, m.desc.vocab)[0])
    m.fork_row(0, 1)
    free = m.get_option("kv.free_tokens")
    k, _ = m.read_kv(0, 0)
    p = k.ctypes.data_as(ctypes.POINTER(ctypes.c_float))
    with pytest.raises(TgxError):
        m._check(m.be.write_kv(m._ctx, 0, 0, None if missing == "keys" else p, None if missing == "values" else p, 300))
    assert m.get_option("kv.free_tokens") == free


@pytest.mark.parametrize("sampler", ["greedy", "sampled"])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("grow", ["fork", "prompt"])
def test_a_pending_token_is_fetched_behind_a_larger_batch(grow, bits, sampler, hip):
    """steps are issued, a row joins the batch, and then their tokens are fetched: those of the same steps without it"""
    cfg = GREEDY if sampler == "greedy" else SamplerCfg(temperature=2.0, top_p=1.0)
    got = []
    for joined in (False, True):
        m, _ = make("llama_tiny", hip, "bf16", bits, max_batch=3, budget=2048)
        p = ids(np.random.default_rng(1), 60, m.desc.vocab)[0]
        m.forward_row(0, p)
        m.sample_row(0, cfg, seed=3)
        tickets = [m.step_async(cfg, seed=3) for _ in range(5)]
        if joined:
            if grow == "fork":
                m.fork_row(0, 1)
            else:
                m.forward_row(1, p[:20])
        got.append([m.fetch_token(t) for t in tickets])
    assert got[0] == got[1] and len(set(got[0])) > 1


# ---- operators -------------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fresh", [False, True])
def test_batches_of_more_than_65535_tokens(fresh):
    """66 prompts of 1000 tokens with max_count left out: what the same call gives where it names 1000, and every prompt alone"""
    from tinygpt_amd import ops
    n, rows, kv, hd, group = 1000, 66, 1, 64, 4
    g = torch.Generator("cuda").manual_seed(1)
    cache = ops.Kv4Cache.empty(1, 8 * rows, kv, hd, rows, n)
    cache.table[:] = torch.randperm(8 * rows, device="cuda", generator=g).int().view(rows, 8)
    k, v, q = (torch.randn(rows * n, h, hd, device="cuda", generator=g).bfloat16() for h in (kv, kv, kv * group))
    start, offsets = ints([0] * rows), ints(range(0, rows * n + 1, n))
    if not fresh:
        ops.kv4_append(cache, k, v, start, offsets=offsets)
    out = ops.kv4_attend(cache, q, start, n, offsets=offsets, **(dict(k=k, v=v) if fresh else {}))
    assert torch.equal(out, ops.kv4_attend(cache, q, start, n, offsets=offsets, max_count=n))
    for i in (0, 40, 65):
        s = slice(i * n, i * n + n)
        one = ops.kv4_attend(cache, q[s], ints([0]), n, seq=ints([i]), offsets=ints([0, n]))
        want = torch.nn.functional.softmax((q[s].double().transpose(0, 1) @ ops.kv4_read(cache, ints([0]), n, seq=ints([i]), offsets=ints([0, n]))[0].double().permute(1, 2, 0).contiguous() / 8)
                                           .masked_fill(~torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), -float("inf")), -1)
        want = (want @ ops.kv4_read(cache, ints([0]), n, seq=ints([i]), offsets=ints([0, n]))[1].double().transpose(0, 1)).transpose(0, 1)
        for o in (out[s], one):      # (divided or not: within the outputs' rounding)
            assert float(((o.double() - want) ** 2).mean()) <= float((2.0 ** -8 * want).square().mean()) / 3 * 1.02


def test_nothing_to_bring_and_nowhere_to_put_it():
    """entries without tokens, a table without pages, a pool without any: outputs of zero for what sees nothing, and no more"""
    from tinygpt_amd import ops
    kv, hd, heads = 2, 64, 4
    full = ops.Kv4Cache.empty(1, 3, kv, hd, 2, 300)
    none, empty = torch.empty(0, kv, hd, device="cuda"), torch.empty(0, heads, hd, device="cuda")
    for e in (1, 3):
        batch = dict(offsets=ints([0] * (e + 1)), seq=ints([0] * e))
        ops.kv4_append(full, none, none, ints([5] * e), **batch)
        assert [t.shape for t in ops.kv4_read(full, ints([5] * e), 0, **batch)] == [none.shape] * 2
        assert ops.kv4_attend(full, empty, ints([5] * e), 300, **batch).shape == empty.shape
        assert ops.kv4_attend(full, empty, ints([5] * e), 300, k=none, v=none, **batch).shape == empty.shape
    q, k = torch.randn(2, heads, hd, device="cuda"), torch.randn(2, kv, hd, device="cuda")
    pool = torch.empty(1, 0, kv * hd * 144, dtype=torch.uint8, device="cuda")
    for cache in (ops.Kv4Cache.empty(1, 3, kv, hd, 2, 0), ops.Kv4Cache(pool, torch.zeros(2, 3, dtype=torch.int32, device="cuda"), kv, hd)):
        start = ints([0, 7])
        ops.kv4_append(cache, k, k, start)
        assert not any(t.any() for t in ops.kv4_read(cache, start, 2))
        assert not ops.kv4_attend(cache, q, start, 8).any() and not ops.kv4_attend(cache, q, start, 8, k=k, v=k).any()
        assert not ops.kv4_attend(cache, q, ints([4]), 8, offsets=ints([0, 2]), k=k, v=k).any()
    assert ops.copy_pages(pool, ints([0, 1]), ints([1, 0])) is pool
    other = torch.full((1, 2, kv * hd * 144), 7, dtype=torch.uint8, device="cuda")
    ops.copy_pages(pool, ints([0, 1]), ints([1, 0]), into=other)
    assert (other == 7).all()


def test_a_generation_finds_its_workspace_again():
    """max_keys grows with every token: the workspace's size is asked of the library once a page of 128"""
    from tinygpt_amd import ops
    cache = ops.Kv4Cache.empty(1, 40, 2, 64, 1, 5000)
    cache.table[0] = torch.arange(cache.table.shape[1], device="cuda").int()
    q, k = torch.randn(1, 8, 64, device="cuda"), torch.randn(1, 2, 64, device="cuda")
    for keys in range(1, 641):
        ops.kv4_attend(cache, q, ints([keys - 1]), keys, k=k, v=k)
        if keys == 1:
            misses = ops._workspace.cache_info().misses
    assert ops._workspace.cache_info().misses - misses <= 4


def test_outputs_that_lie_on_each_other_are_refused():
    from tinygpt_amd import ops
    cache = ops.Kv4Cache.empty(1, 4, 2, 64, 2, 300)
    cache.table[:] = ints(range(4)).view(2, 2).repeat(1, 2)[:, :cache.table.shape[1]]
    q, start = torch.randn(2, 4, 64, device="cuda"), ints([0, 5])
    k = torch.randn(1, 2, 64, device="cuda").expand(2, 2, 64)      # the same token twice: an input may
    ops.kv4_append(cache, k, k, start)
    for shape in [(1, 4, 64), (2, 1, 64), (1, 1, 64)]:
        with pytest.raises(TgxError):
            ops.kv4_attend(cache, q, start, 300, out=torch.zeros(shape, device="cuda").expand(2, 4, 64))
    with pytest.raises(TgxError):
        ops.kv4_read(cache, start, 2, out=(torch.zeros(2, 2, 64, device="cuda"), torch.zeros(1, 2, 64, device="cuda").expand(2, 2, 64)))
    one = torch.zeros(1, 4, 64, device="cuda")
    ops.kv4_attend(cache, q[:1], start[:1], 300, out=one.as_strided((1, 4, 64), (0, 64, 1)))      # one token: its stride says nothing
    assert torch.equal(one, ops.kv4_attend(cache, q[:1], start[:1], 300)) and one.any()


def test_copies_into_layers_that_share_memory_are_refused():
    from tinygpt_amd import ops
    pool = torch.randint(0, 99, (1, 4, 64), device="cuda", dtype=torch.int32)
    with pytest.raises(TgxError):
        ops.copy_pages(torch.zeros(3, 4, 64, device="cuda", dtype=torch.int32), ints([0]), ints([1]), into=pool.expand(3, 4, 64))
    into = torch.zeros(3, 4, 64, device="cuda", dtype=torch.int32)
    ops.copy_pages(pool.expand(3, 4, 64), ints([2, 0]), ints([1, 3]), into=into)      # one layer into three
    assert torch.equal(into[:, [1, 3]], pool[:, [2, 0]].expand(3, 2, 64)) and not into[:, [0, 2]].any()
    wide = torch.zeros(3, 6, 64, device="cuda", dtype=torch.int32)                    # pages of a larger pool: layers further apart than their pages
    ops.copy_pages(pool.expand(3, 4, 64), ints([2, 0]), ints([1, 3]), into=wide[:, 1:5])
    assert torch.equal(wide[:, [2, 4]], pool[:, [2, 0]].expand(3, 2, 64)) and not wide[:, [0, 1, 3, 5]].any()


def test_a_read_of_positions_that_are_not_there():
    """negative positions are left as they were, positions without a page read as zeros, in every type and by tokens and portions"""
    from tinygpt_amd import ops
    for dtype in (torch.bfloat16, torch.float32):
        cache = ops.Kv4Cache.empty(1, 3, 2, 64, 1, 300)
        cache.table[0, 0] = 2      # and no second page
        x = torch.randn(128, 2, 64, device="cuda").to(dtype)
        ops.kv4_append(cache, x, x, ints([0]), offsets=ints([0, 128]))
        k, v = torch.full((2, 160, 2, 64), 7.0, dtype=dtype, device="cuda").unbind(0)
        ops.kv4_read(cache, ints([-10]), 160, offsets=ints([0, 160]), out=(k, v))
        for t in (k, v):
            assert (t[:10] == 7).all() and not t[138:].any() and (t[10:138] - x).abs().max() < 0.5
            assert torch.equal(t[10:138], ops.kv4_read(cache, ints([0]), 128, dtype=dtype, offsets=ints([0, 128]))[0])
        one = torch.full((2, 1, 2, 64), 7.0, dtype=dtype, device="cuda")
        ops.kv4_read(cache, ints([-1]), 1, out=one.unbind(0))
        assert (one == 7).all()
