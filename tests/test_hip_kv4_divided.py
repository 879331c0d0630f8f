"""Models over a 4-bit cache whose steps divide the keys between workgroups (from 2048 keys on at head_dim 64, 1024 at 128) or run in several parts: records, their workspace, graphs on both sides
of a division."""
import numpy as np
import pytest

from test_hip_kv4_model import Stepper, ids, make, near
from tinygpt_amd.ffi import GREEDY

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from tinygpt_amd.ffi import product_backend
    return product_backend()


@pytest.mark.parametrize("fam", ["llama_tiny", "mistral_tiny", "qwen2_tiny"])      # head_dim 64, 128 and, without shared heads, 64
@pytest.mark.parametrize("batch,n", [(1, 1020), (1, 1500), (1, 2046), (3, 2090), (6, 2090)])
def test_steps_over_divided_keys(fam, batch, n, hip):
    """a step's logits against the model's equations in 64 bits over what the cache holds, within 1e-3 of the largest; the equations without the values of one page of 128 tokens, or of
    the 32 in front of the step's, are further off than that"""
    m, g = make(fam, hip, "bf16", 4, max_batch=batch, max_ctx=4096, budget=(n + 300) * batch)
    ref = Stepper(m.desc, int(g["seed"]), float(g["std"]))
    m.forward(ids(np.random.default_rng(7), n, m.desc.vocab, batch))
    toks = m.sample(GREEDY)
    for step in range(3):
        after = m.decode(1)[0]
        got = m.logits(rounded=False)
        for row in range(batch):
            cache = [m.read_kv(row, layer) for layer in range(m.desc.layers)]
            near(got[row], ref.logits(int(toks[row]), cache), 1e-3)
            if step == 0 and row == 0:
                for a, b in [(0, 128), (512, 640), (n - 32, n)]:
                    lost = [(k, np.concatenate([v[:a], 0 * v[a:b], v[b:]])) for k, v in cache]
                    with pytest.raises(AssertionError):
                        near(got[row], ref.logits(int(toks[row]), lost), 1e-3)
        toks = after


@pytest.mark.parametrize("fam,n,steps", [("llama_tiny", 2000, 110), ("mistral_tiny", 980, 100)])
@pytest.mark.parametrize("batch,act", [(1, 0), (2, 1), (5, 0), (8, 1)])
def test_graphs_on_both_sides_of_a_division(fam, n, steps, batch, act, hip):
    """a generation across the key counts at which the keys come to be divided, in graphs of many steps and one step at a time without: the same tokens, the same bits"""
    ms = []
    for graph in (1, 0):
        m, _ = make(fam, hip, "bf16", 4, max_batch=batch, max_ctx=4096, budget=(n + steps + 200) * batch, opts=(("graph", graph), ("act.round16", act)))
        m.forward(ids(np.random.default_rng(11), n, m.desc.vocab, batch))
        first = m.sample(GREEDY)
        ms.append((m, first, m.decode(steps) if graph else np.concatenate([m.decode(1) for _ in range(steps)])))
    (a, fa, ta), (b, fb, tb) = ms
    assert (fa == fb).all() and (ta == tb).all()
    assert np.array_equal(a.logits(rounded=False), b.logits(rounded=False))
    for row in range(batch):
        for x, y in zip(a.read_kv(row, 1), b.read_kv(row, 1)):
            assert np.array_equal(x, y)


@pytest.mark.parametrize("batch,opts", [(40, ()), (40, (("decode.step_rows", 64),)), (9, ())])
def test_steps_in_several_parts(batch, opts, hip):
    """more rows than a pass over the weights takes: every part's rows attend to their own pages"""
    m, g = make("llama_tiny", hip, "bf16", 4, max_batch=batch, max_ctx=512, budget=256 * batch, opts=opts)
    ref = Stepper(m.desc, int(g["seed"]), float(g["std"]))
    m.forward(ids(np.random.default_rng(7), 130, m.desc.vocab, batch))
    toks = m.sample(GREEDY)
    for _ in range(2):
        after = m.decode(1)[0]
        got = m.logits(rounded=False)
        for row in sorted({0, 7, 8, 31, 32, batch - 1} & set(range(batch))):
            near(got[row], ref.logits(int(toks[row]), [m.read_kv(row, layer) for layer in range(m.desc.layers)]), 1e-3)
        toks = after
