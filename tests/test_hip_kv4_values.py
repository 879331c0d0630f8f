"""Values of attention over a 4-bit cache (tinygpt_amd.ops) near 64 bits, as near as kv4_near.py derives: short and long walks, divided and whole, every form."""
import numpy as np
import pytest
import torch   # here, not in a test: before any module's test loads the library, which then shares torch's HIP runtime

from kv4_near import STEP

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


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
