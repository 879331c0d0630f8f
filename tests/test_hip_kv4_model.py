"""Models over a cache in 4 bits (option kv.bits 4), rows that are forked and pools that are resized (tgx_fork_row, tgx_resize_kv).

A prompt runs on the same kernels as over a 16-bit cache and leaves exactly the levels of the same keys and values; a step is held to the model's equations in 64 bits over the values that
the cache holds."""
import numpy as np
import pytest

from conftest import load_golden
from kv4_util import values
from tinygpt_amd import synth
from tinygpt_amd.desc import desc_from_hf_config
from tinygpt_amd.ffi import GREEDY, Model, SamplerCfg, TgxError

pytestmark = pytest.mark.gpu
CONTEXT, STATE, UNSUPPORTED, INVALID = 8, 4, 2, 1


@pytest.fixture(scope="module")
def hip():
    from tinygpt_amd.ffi import product_backend
    return product_backend()


def make(fam, hip, dtype="fp16", bits=16, max_batch=2, max_ctx=512, budget=1024, opts=(), scale=1.0):
    cfg, g = load_golden(fam)
    d = desc_from_hf_config(cfg, dtype, max_batch=max_batch)
    d.max_ctx = min(max_ctx, d.max_ctx) if fam.startswith("gpt2") else max_ctx
    if fam.startswith("gpt2"):
        d.max_ctx = min(max_ctx, d.n_positions)
    m = Model(d, hip)
    m.set_option("kv.budget_tokens", budget)
    if bits != 16:
        m.set_option("kv.bits", bits)
    m.load_synthetic(int(g["seed"]), float(g["std"])).finalize()
    for k, v in opts:
        m.set_option(k, v)
    return m, g


def ids(rng, n, vocab, rows=1):
    return rng.integers(0, vocab, (rows, n))


def held(x):
    return values(x)[0].astype(np.float32)


def near(a, b, tol):
    err = float(np.abs(a - b).max() / np.abs(b).max())
    assert err < tol, err


FAMS = [("llama_tiny", "fp16"), ("llama_tiny", "bf16"), ("qwen2_tiny", "fp16"), ("mistral_tiny", "bf16"), ("qwen3_tiny", "fp16"), ("gpt2_hd64", "fp16")]


@pytest.mark.parametrize("fam,dtype", FAMS)
@pytest.mark.parametrize("n", [1, 3, 5, 40, 129])
def test_prompts_leave_the_levels_of_their_keys_and_values(fam, dtype, n, hip):
    """by steps (short prompts), on the skinny products and on the tiles; the keys and values of the 16-bit cache are what is quantised: bit for bit where a pass attends to what it computed"""
    a, g = make(fam, hip, dtype, 4)
    b, _ = make(fam, hip, dtype, 16)
    if n > a.desc.max_ctx - 4:
        pytest.skip("beyond this fixture's context")
    p = ids(np.random.default_rng(n), n, a.desc.vocab, 2)
    a.forward(p); b.forward(p)
    layers = range(a.desc.layers) if n >= 5 else [0]      # a prompt by steps attends to the quantised cache: only the first layer's inputs are the same
    for layer in layers:
        for row in range(2):
            for got, src in zip(a.read_kv(row, layer), b.read_kv(row, layer)):
                assert np.array_equal(got, held(src)), (layer, row)
    if n >= 5:
        assert np.array_equal(a.logits(rounded=False), b.logits(rounded=False))


def rope_angles(d, pos):
    """angles of a position's pairs, with Llama 3's scaling where the model has it"""
    half = d.head_dim // 2
    inv = d.rope_theta ** (-2.0 * np.arange(half) / d.head_dim)
    if d.rope_factor > 0:
        wl = 2 * np.pi / inv
        low, high = d.rope_orig_ctx / d.rope_low_freq, d.rope_orig_ctx / d.rope_high_freq
        v = np.where(wl > low, inv / d.rope_factor, inv)
        sm = (d.rope_orig_ctx / wl - d.rope_low_freq) / (d.rope_high_freq - d.rope_low_freq)
        inv = np.where((wl >= high) & (wl <= low), (1 - sm) * v / d.rope_factor + sm * v, v)
    return pos * inv


class Stepper:
    """logits of one token at the end of a row whose keys and values (this token's among them) are given, in 64 bits"""

    def __init__(self, d, seed, std):
        self.d, self.w = d, {n: synth.bf16_bits_to_f32(b).astype(np.float64) for n, b in synth.synth_checkpoint(d, seed, std, False)}

    def logits(self, token, cache):
        d, w = self.d, self.w
        D, G, pos = d.head_dim, d.heads // d.kv_heads, len(cache[0][0]) - 1

        def norm(v, n):
            return v / np.sqrt((v * v).mean(-1, keepdims=True) + d.norm_eps) * w[n]

        x = w["model.embed_tokens.weight"][token]
        for i in range(d.layers):
            p = "model.layers.%d." % i
            h = norm(x, p + "input_layernorm.weight")
            q = (w[p + "self_attn.q_proj.weight"] @ h + (w[p + "self_attn.q_proj.bias"] if d.qkv_bias else 0)).reshape(d.heads, D)
            if d.qk_norm:
                q = norm(q, p + "self_attn.q_norm.weight")
            a = rope_angles(d, pos)
            lo, hi = q[:, :D // 2], q[:, D // 2:]
            q = np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)], 1)
            k, v = (t.astype(np.float64) for t in cache[i])
            o = np.zeros((d.heads, D))
            for hd in range(d.heads):
                s = k[:, hd // G] @ q[hd] / np.sqrt(D)
                e = np.exp(s - s.max())
                o[hd] = e @ v[:, hd // G] / e.sum()
            x = x + w[p + "self_attn.o_proj.weight"] @ o.reshape(-1)
            h = norm(x, p + "post_attention_layernorm.weight")
            g = w[p + "mlp.gate_proj.weight"] @ h
            x = x + w[p + "mlp.down_proj.weight"] @ (g / (1 + np.exp(-g)) * (w[p + "mlp.up_proj.weight"] @ h))
        head = w["model.embed_tokens.weight"] if d.tied else w["lm_head.weight"]
        return head @ norm(x, "model.norm.weight")


@pytest.mark.parametrize("fam", ["llama_tiny", "qwen2_tiny", "qwen3_tiny", "mistral_tiny"])
@pytest.mark.parametrize("batch,n", [(1, 130), (1, 400), (2, 130), (4, 130), (6, 130)])
def test_steps_attend_to_what_the_cache_holds(fam, batch, n, hip):
    """a step's logits against the model's equations in 64 bits over the keys and values that the cache holds afterwards, the step's own among them: within 1e-3 of the largest, as all
    logits of the 16-bit models are held to their oracle"""
    m, g = make(fam, hip, "bf16", 4, max_batch=batch, budget=512 * batch)
    ref = Stepper(m.desc, int(g["seed"]), float(g["std"]))
    m.forward(ids(np.random.default_rng(7), n, m.desc.vocab, batch))
    toks = m.sample(GREEDY)
    for step in range(2):
        after = m.decode(1)[0]
        got = m.logits(rounded=False)
        for row in range(batch):
            near(got[row], ref.logits(int(toks[row]), [m.read_kv(row, layer) for layer in range(m.desc.layers)]), 1e-3)
        toks = after


@pytest.mark.parametrize("fam", ["llama_tiny", "gpt2_hd64"])
def test_prompts_by_steps_attend_to_what_the_cache_holds(fam, hip):
    """several positions of a sequence a pass: each reads what the pass itself appends"""
    a, g = make(fam, hip, "bf16", 4, max_batch=1, opts=(("prefill.mfma", 0),))
    n = min(150, a.desc.max_ctx - 4)
    p = ids(np.random.default_rng(4), n, a.desc.vocab)
    a.forward(p[:, :n])
    b, _ = make(fam, hip, "bf16", 4, max_batch=1, opts=(("prefill.mfma", 0),))
    b.forward(p[:, :1])
    for i in range(1, n):      # one by one
        b.forward(p[:, i:i + 1])
    assert np.array_equal(a.logits(rounded=False), b.logits(rounded=False))
    for layer in range(a.desc.layers):
        for x, y in zip(a.read_kv(0, layer), b.read_kv(0, layer)):
            assert np.array_equal(x, y)
    if fam == "llama_tiny":
        near(a.logits(rounded=False)[0], Stepper(a.desc, int(g["seed"]), float(g["std"])).logits(int(p[0, -1]), [a.read_kv(0, layer) for layer in range(a.desc.layers)]), 1e-3)


@pytest.mark.parametrize("batch,opts", [(1, ()), (1, (("graph", 0),)), (2, ()), (3, (("act.round16", 1),)), (8, ())])
def test_long_generations_are_their_own_steps(batch, opts, hip):
    """graphs of many steps across the limits at which the keys are divided anew (256, 512), against steps one by one without graphs: the same tokens and the same bits in the cache"""
    ms = []
    for graph in (1, 0):
        m, g = make("llama_tiny", hip, "bf16", 4, max_batch=batch, max_ctx=768, budget=768 * batch, opts=tuple(opts) + (("graph", graph),) if not opts or opts[0][0] != "graph" else opts)
        p = ids(np.random.default_rng(11), 230, m.desc.vocab, batch)
        m.forward(p)
        first = m.sample(GREEDY)
        toks = m.decode(310) if graph else np.concatenate([m.decode(1) for _ in range(310)])
        ms.append((m, first, toks))
    assert (ms[0][1] == ms[1][1]).all() and (ms[0][2] == ms[1][2]).all()
    assert np.array_equal(ms[0][0].logits(rounded=False), ms[1][0].logits(rounded=False))
    for row in range(batch):
        for x, y in zip(ms[0][0].read_kv(row, 1), ms[1][0].read_kv(row, 1)):
            assert np.array_equal(x, y)


def test_rows_come_and_go(hip):
    """rows of a batch of unequal lengths, one retired and refilled while the others step: each as alone"""
    m, g = make("llama_tiny", hip, "bf16", 4, max_batch=3, budget=1024)
    rng = np.random.default_rng(2)
    prompts = [ids(rng, n, m.desc.vocab)[0] for n in (150, 40, 7)]
    for r, p in enumerate(prompts):
        m.forward_row(r, p)
        m.sample_row(r)
    m.decode(20)
    m.reset_row(1)
    m.decode(5)
    late = ids(rng, 60, m.desc.vocab)[0]
    m.forward_row(1, late)
    first = m.sample_row(1)
    toks = m.decode(10)
    alone, _ = make("llama_tiny", hip, "bf16", 4, max_batch=3, budget=1024)
    for r, p in enumerate([late, late, late]):      # (the same batch size: the same kernels)
        alone.forward_row(r, p)
        assert alone.sample_row(r) == first
    assert (alone.decode(10)[:, 0] == toks[:, 1]).all()


# ---- forks ----------------------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("n", [5, 127, 128, 129, 300])
def test_a_fork_goes_on_as_its_source(bits, n, hip):
    m, g = make("llama_tiny", hip, "bf16", bits, max_batch=4, budget=2048)
    p = ids(np.random.default_rng(n), n, m.desc.vocab)[0]
    m.forward_row(0, p)
    free = m.get_option("kv.free_tokens")
    m.fork_row(0, 1)                                      # before its first token: n samples of one prompt
    assert m.get_option("kv.free_tokens") == free - (128 if n % 128 else 0)
    assert np.array_equal(m.logits()[0], m.logits()[1])
    for layer in range(m.desc.layers):
        for x, y in zip(m.read_kv(0, layer), m.read_kv(1, layer)):
            assert np.array_equal(x, y)
    assert m.sample_row(0) == m.sample_row(1)
    both = m.decode(9)
    assert (both[:, 0] == both[:, 1]).all() and np.array_equal(m.logits()[0], m.logits()[1])
    m.fork_row(1, 2)                                      # behind its token
    three = m.decode(7)
    assert (three[:, 0] == three[:, 2]).all() and m.past_length_row(2) == n + 16
    # rows that part keep their own: another token in row 2
    cfg = SamplerCfg(temperature=5.0, top_p=1.0)
    m.sample_row(2, cfg, seed=5)
    before = [m.read_kv(0, layer)[0][:n].copy() for layer in range(m.desc.layers)]
    m.decode(130)
    for layer in range(m.desc.layers):
        assert np.array_equal(m.read_kv(0, layer)[0][:n], before[layer]) and np.array_equal(m.read_kv(2, layer)[0][:n], before[layer])
    got = m.read_kv(0, 0)[0]
    # the source goes, the forks stay
    m.reset_row(0)
    assert np.array_equal(m.read_kv(1, 0)[0][:n], got[:n])
    m.reset_row(1); m.reset_row(2)
    assert m.get_option("kv.free_tokens") == 2048


def test_forked_rows_against_rows_of_their_own(hip):
    """a fork and its source, each with a different continuation, against two prompts prefilled one by one with those continuations decoded"""
    m, g = make("qwen2_tiny", hip, "bf16", 16, max_batch=2, budget=1024)
    p = ids(np.random.default_rng(1), 200, m.desc.vocab)[0]
    cfg = SamplerCfg(temperature=3.0, top_p=1.0)
    m.forward_row(0, p)
    m.fork_row(0, 1)
    t = [m.sample_row(0, cfg, seed=1), m.sample_row(1, cfg, seed=2)]
    toks = m.decode(40)
    w, _ = make("qwen2_tiny", hip, "bf16", 16, max_batch=2, budget=1024)
    w.forward_row(0, p); w.forward_row(1, p)
    assert [w.sample_row(0, cfg, seed=1), w.sample_row(1, cfg, seed=2)] == t
    assert (w.decode(40) == toks).all() and np.array_equal(w.logits(), m.logits())


def test_writes_to_a_row_leave_its_fork(hip):
    for bits in (16, 4):
        m, g = make("llama_tiny", hip, "bf16", bits, max_batch=2, budget=1024)
        m.forward_row(0, ids(np.random.default_rng(1), 300, m.desc.vocab)[0])
        m.fork_row(0, 1)
        k, v = m.read_kv(1, 1)
        m.write_kv(0, 1, np.zeros_like(k), np.zeros_like(v))
        for x, y in zip(m.read_kv(1, 1), (k, v)):
            assert np.array_equal(x, y)
        assert not m.read_kv(0, 1)[0].any()


def test_fork_refusals(hip):
    m, g = make("llama_tiny", hip, "bf16", 4, max_batch=3, budget=384)

    def refused(status, f):
        with pytest.raises(TgxError) as e:
            f()
        assert e.value.status == status, e.value

    refused(INVALID, lambda: m.fork_row(0, 1))            # nothing there
    m.forward_row(0, ids(np.random.default_rng(1), 290, m.desc.vocab)[0])
    for src, dst, status in [(0, 0, INVALID), (0, 2, INVALID), (0, -1, INVALID), (0, 3, INVALID), (1, 2, INVALID), (-1, 1, INVALID)]:
        refused(status, lambda: m.fork_row(src, dst))
    refused(CONTEXT, lambda: m.fork_row(0, 1))            # all three blocks in use, a fork needs one
    assert m.past_length_row(0) == 290 and m.past_length_row(1) == 0
    m.sample_row(0)
    m.decode(3)                                           # and nothing has changed
    m.resize_kv(512)
    m.fork_row(0, 1)
    refused(STATE, lambda: m.fork_row(0, 1))              # a live row is reset first
    m.reset_row(0)
    refused(INVALID, lambda: m.fork_row(0, 2))            # a retired one holds nothing
    cfg, g = load_golden("llama_tiny")
    d = desc_from_hf_config(cfg, "bf16", max_batch=2)
    flat = Model(d, hip).load_synthetic(int(g["seed"]), float(g["std"])).finalize()
    flat.forward(ids(np.random.default_rng(1), 9, d.vocab))
    refused(UNSUPPORTED, lambda: flat.fork_row(0, 1))
    refused(UNSUPPORTED, lambda: flat.resize_kv(512))


# ---- pools made larger and smaller ----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [16, 4])
def test_a_resized_pool_keeps_its_rows(bits, hip):
    m, g = make("llama_tiny", hip, "bf16", bits, max_batch=3, max_ctx=768, budget=1536)
    w, _ = make("llama_tiny", hip, "bf16", bits, max_batch=3, max_ctx=768, budget=1536)
    rng = np.random.default_rng(5)
    for r, n in enumerate((300, 90, 200)):
        p = ids(rng, n, m.desc.vocab)[0]
        for x in (m, w):
            x.forward_row(r, p)
            x.sample_row(r)
    for x in (m, w):
        x.decode(10)
        x.reset_row(1)                                   # holes in the pool
    m.resize_kv(640)                                      # 3 + 2 blocks, none free
    assert m.get_option("kv.free_tokens") == 0 and m.get_option("kv.budget_tokens") == 640
    with pytest.raises(TgxError) as e:
        m.resize_kv(512)                                  # four blocks (600 tokens would still be five)
    assert e.value.status == CONTEXT
    for layer in range(m.desc.layers):
        for row in (0, 2):
            for x, y in zip(m.read_kv(row, layer), w.read_kv(row, layer)):
                assert np.array_equal(x, y)
    assert (m.decode(40)[:, [0, 2]] == w.decode(40)[:, [0, 2]]).all()
    with pytest.raises(TgxError) as e:
        m.decode(100)                                     # beyond the last block
    assert e.value.status == CONTEXT
    m.resize_kv(2048)
    a, b = m.decode(150), w.decode(150)
    assert (a[:, [0, 2]] == b[:, [0, 2]]).all()
    m.fork_row(0, 1)
    m.resize_kv(1280)                                     # shared blocks stay shared
    assert (m.decode(5)[:, 0] == w.decode(5)[:, 0]).all()
    assert np.array_equal(m.read_kv(0, 1)[0], m.read_kv(1, 1)[0])
    for r in range(3):
        m.reset_row(r)
    assert m.get_option("kv.free_tokens") == 1280
    m.resize_kv(128)
    m.forward_row(0, ids(rng, 100, m.desc.vocab)[0])
    assert m.get_option("kv.free_tokens") == 0


def test_options(hip):
    cfg, g = load_golden("llama_tiny")
    d = desc_from_hf_config(cfg, "bf16", max_batch=1)

    def refused(status, f):
        with pytest.raises(TgxError) as e:
            f()
        assert e.value.status == status, e.value

    m = Model(d, hip)
    refused(INVALID, lambda: m.set_option("kv.bits", 8))
    m.set_option("kv.bits", 4)
    assert m.get_option("kv.bits") == 4
    m.load_synthetic(int(g["seed"]), float(g["std"]))
    refused(UNSUPPORTED, m.finalize)                      # without a paged cache
    m.set_option("kv.budget_tokens", 256)
    m.finalize()
    refused(STATE, lambda: m.set_option("kv.bits", 16))
    m.forward(ids(np.random.default_rng(1), 20, d.vocab))
    k, v = m.read_kv(0, 0)
    with pytest.raises(TgxError):
        m._check(m.be.write_kv(m._ctx, 0, 0, k.ctypes.data_as(__import__("ctypes").POINTER(__import__("ctypes").c_float)), None, 3))
    f = Model(desc_from_hf_config(cfg, "fp32", max_batch=1), hip)
    refused(UNSUPPORTED, lambda: f.set_option("kv.bits", 4))
    per = m.desc.layers * m.desc.kv_heads * m.desc.head_dim
    assert m.be.bytes_per_token(m._ctx, 800) - m.be.bytes_per_token(m._ctx, 0) == per * 900
