"""The operators of a cache held in 4 bits, as calls that can be timed and compared: attention of single tokens and of portions over it, the append that fills
it, and the copies that fork rows and compact pools.

  listed()                  the cases, each with what it stands for beside it
  draw(rng)                 one more case of the same ranges
  prepare(case, seed)       pages, page table, queries, keys and values on the GPU: what a program holds before the call
  run(state)                one pass: in elementary torch operations, or (own = True) through tinygpt_amd.ops
  exact(case, seed)         the same outputs in 64 bits
  work(case)                bytes and operations that a pass cannot do without

The cache.  A page holds 128 tokens of all key / value heads; page 0 takes the writes of table entries without a page.  64 neighbouring channels of a token
and head are a group: 16 levels lo + step * n, lo and step in bfloat16, n in 4 bits.
  lo = min x rounded down to bfloat16, step = max((max x - lo) * (1 / 15) rounded up to bfloat16, 2^-126), n = min(15, rint((x - lo) * (1 / step)))
with every operation rounded to 32 bits.  A page's head is four blocks of 32 tokens, each of 16 * dim bytes of key codes, 16 * dim bytes of value codes and
4 * dim bytes of parameters.  Codes lie in 32-bit words of eight, in the order in which the matrix cores of the GPU take them:
  key word ((part * 64 + 16 q + r) * 4 + w), i = 4 part + w: token 16 (i // (dim / 32)) + r, channels 32 (i % (dim / 32)) + 8 q + e
  value word ((part * 64 + 16 q + r) * 4 + w):               channel 16 (4 part + w) + r, tokens 4 q + e (e < 4) and 12 + 4 q + e
e = 0 .. 7 in the bits from 4 * (e // 2 + 4 * (e % 2)) on.  Parameters: [32 tokens][keys, values][dim / 64], lo in the low half of a word, step in the high.
"""
import math

import torch

own = False

PAGE = 128
TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one stream of a small model: the next token of a chat, where latency is what counts
        dict(name="token-chat", kind="attend", seqs=1, ctx=713, ragged=False, count=1, heads=32, kv_heads=8, dim=64, dtype="bf16", window=0, fresh=False),
        # three short rows of a model without shared heads, in 32 bits; the tokens' keys and values join the cache in the same call
        dict(name="tokens-gpt2-fp32", kind="attend", seqs=3, ctx=261, ragged=True, count=1, heads=12, kv_heads=12, dim=64, dtype="fp32", window=0, fresh=True),
        # a running batch of a small model, seven query heads a key / value head
        dict(name="tokens-batch-fp16", kind="attend", seqs=64, ctx=1500, ragged=True, count=1, heads=14, kv_heads=2, dim=64, dtype="fp16", window=0, fresh=False),
        # a running batch of a larger model, one step of it: append and attend
        dict(name="tokens-batch", kind="attend", seqs=32, ctx=4096, ragged=True, count=1, heads=32, kv_heads=8, dim=128, dtype="bf16", window=0, fresh=True),
        # one stream over the longest context that a model of the framework takes
        dict(name="token-long", kind="attend", seqs=1, ctx=131071, ragged=False, count=1, heads=64, kv_heads=8, dim=128, dtype="bf16", window=0, fresh=False),
        # long rows of which a sliding window shows the end
        dict(name="tokens-window-fp32", kind="attend", seqs=8, ctx=30000, ragged=True, count=1, heads=32, kv_heads=8, dim=128, dtype="fp32", window=4096, fresh=False),
        # proposed tokens of a batch checked in one step: a few a row
        dict(name="proposals", kind="attend", seqs=16, ctx=2000, ragged=True, count=5, heads=16, kv_heads=8, dim=128, dtype="bf16", window=0, fresh=True),
        # the last portion of a long prompt
        dict(name="portion", kind="attend", seqs=1, ctx=8192, ragged=False, count=2048, heads=32, kv_heads=8, dim=128, dtype="bf16", window=0, fresh=True),
        # prompts of several rows join the cache and are read back for a pass that wants the values themselves
        dict(name="append-prompts", kind="append", seqs=4, ctx=4096, ragged=True, count=4096, kv_heads=8, dim=128, dtype="bf16"),
        # a step's tokens of a batch join theirs
        dict(name="append-tokens-fp16", kind="append", seqs=64, ctx=900, ragged=True, count=1, kv_heads=8, dim=64, dtype="fp16"),
        # a row is forked: its last page, in every layer of a 16-bit cache
        dict(name="fork-page", kind="copy", layers=16, pages=40, moved=1, kv_heads=8, dim=64, bits=16),
        # a pool is compacted: pages of many rows move to its front, in every layer of a 4-bit cache
        dict(name="compact-pool", kind="copy", layers=32, pages=400, moved=180, kv_heads=8, dim=128, bits=4),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["attend", "attend", "attend", "append", "copy"])
    heads, kv_heads, dim = rng.choice([(32, 8, 64), (12, 12, 64), (14, 2, 64), (32, 8, 128), (64, 8, 128), (16, 8, 128), (16, 16, 64), (16, 1, 128)])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "copy":
        c = dict(kind=kind, layers=rng.randint(1, 32), kv_heads=kv_heads, dim=dim, bits=rng.choice([4, 16]))
        c["pages"] = size(2, max(2, min(400, 1800000000 // (c["layers"] * page_bytes(c)))))
        return dict(c, moved=rng.randint(1, max(1, c["pages"] * 9 // 20)))
    seqs = rng.choice([1, 1, 2, 3, 7, 16, 33, 64])
    ragged = seqs > 1 and rng.random() < 0.8
    if kind == "append":
        count = rng.choice([1, size(1, 8000 // seqs)])
        return dict(kind=kind, seqs=seqs, ctx=count + rng.choice([0, size(1, 3000)]), ragged=ragged, count=count, kv_heads=kv_heads, dim=dim, dtype=dtype)
    count = rng.choice([1, 1, 1, size(2, 16), size(17, 900)])
    most = (131072 if seqs == 1 else 65536) // seqs if count <= 16 else 8192 // seqs
    count = min(count, most)
    return dict(kind=kind, seqs=seqs, ctx=size(count, most), ragged=ragged, count=count, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                window=rng.choice([0, 0, 0, size(16, 4096)]), fresh=rng.random() < 0.5)


def lengths(case):
    """(tokens after the call, tokens that the call brings) of every row: from a third to the whole of the sizes, from the sizes alone"""
    n, c, k = case["seqs"], case["ctx"], case["count"]
    if not case["ragged"]:
        return [(c, k)] * n
    brought = [max(1, k - (2 * k // 3) * i // max(1, n - 1)) for i in range(n)]
    return [(max(b, c - (2 * c // 3) * i // max(1, n - 1) - (i % 3 if i else 0)), b) for i, b in enumerate(brought)]


# ---- the format --------------------------------------------------------------------------------------------------------------------------------
def page_bytes(case):
    return PAGE * case["kv_heads"] * case["dim"] * 9 // 8 if case.get("bits", 4) == 4 else PAGE * case["kv_heads"] * case["dim"] * 4


def order(dim, values, device):
    """place in a block's [32 tokens][dim] codes of the code at bits 4 j of word i, as [i][j]"""
    i = torch.arange(4 * dim, device=device)[:, None]
    j = torch.arange(8, device=device)[None]
    lane, word, e = i // 4 % 64, i // 256 * 4 + i % 4, 2 * (j % 4) + j // 4
    q, r = lane // 16, lane % 16
    if values:
        token, channel = 4 * q + e + torch.where(e < 4, 0, 12), 16 * word + r
    else:
        token, channel = 16 * (word // (dim // 32)) + r, 32 * (word % (dim // 32)) + 8 * q + e
    return token * dim + channel


def quantise(x):
    """codes, lo, step [..][dim / 64][..] of x [..][dim], in 32 bits"""
    g = x.float().unflatten(-1, (-1, 64))
    low = g.amin(-1, keepdim=True)
    lo = low.view(torch.int32)
    lo = torch.where(low < 0, lo + 0xFFFF, lo).bitwise_and(-65536).view(torch.float32)
    spread = g.amax(-1, keepdim=True) - lo
    step = (spread * torch.tensor(1 / 15, dtype=torch.float32, device=x.device)).view(torch.int32)
    step = (step + 0xFFFF).bitwise_and(-65536).view(torch.float32).clamp(min=2.0 ** -126)
    fine = torch.isfinite(spread)
    n = torch.round((g - lo) * (1 / step)).clamp(max=15)
    n = torch.where(fine, n, torch.zeros_like(n)).to(torch.uint8)
    return n.flatten(-2), torch.where(fine, lo, torch.full_like(lo, math.nan))[..., 0], torch.where(fine, step, torch.zeros_like(step))[..., 0]


def pack(codes, dim, values):
    """codes [..][32][dim] as words [..][4 dim]"""
    c = codes.flatten(-2)[..., order(dim, values, codes.device)].to(torch.int32)
    return (c << (4 * torch.arange(8, device=c.device, dtype=torch.int32))).sum(-1, dtype=torch.int64).to(torch.int32)


def unpack(words, dim, values):
    c = (words[..., None] >> (4 * torch.arange(8, device=words.device, dtype=torch.int32))).bitwise_and(15).to(torch.uint8).flatten(-2)
    place = torch.empty(32 * dim, dtype=torch.int64, device=words.device)
    place[order(dim, values, words.device).flatten()] = torch.arange(32 * dim, device=words.device)
    return c[..., place].unflatten(-1, (32, dim))


def pages_of(codes, lo, step, dim):
    """words [pages][kv_heads][block][9 dim] of codes [2][pages][128][kv_heads][dim] and their parameters [2][pages][128][kv_heads][dim / 64]"""
    c = codes.transpose(2, 3).unflatten(3, (4, 32))
    p = (step.view(torch.int32).bitwise_and(-65536) | (lo.view(torch.int32) >> 16).bitwise_and(0xFFFF)).transpose(2, 3).unflatten(3, (4, 32))
    p = p.permute(1, 2, 3, 4, 0, 5).flatten(-3)
    return torch.cat([pack(c[0], dim, False), pack(c[1], dim, True), p], -1)


def parts_of(words, dim):
    """the inverse of pages_of, with any number of leading sizes in the place of the pages"""
    k, v, p = words.split([4 * dim, 4 * dim, dim], -1)
    c = torch.stack([unpack(k, dim, False), unpack(v, dim, True)]).flatten(-3, -2).transpose(-3, -2)
    p = p.unflatten(-1, (32, 2, dim // 64)).movedim(-2, 0).flatten(-3, -2).transpose(-3, -2)
    return c, (p << 16).view(torch.float32), p.bitwise_and(-65536).view(torch.float32)


def value_of(codes, lo, step):
    return (lo[..., None] + step[..., None] * codes.unflatten(-1, (-1, 64)).to(lo.dtype)).flatten(-2)


# ---- what a program holds ------------------------------------------------------------------------------------------------------------------------
def rows_of(case, seed):
    """keys and values [2][tokens of all rows][kv_heads][dim] in the storage type, queries of the tokens that the call brings, and where they lie"""
    g = torch.Generator("cuda").manual_seed(seed * 7919 + 17)
    H, D, t = case["kv_heads"], case["dim"], TORCH[case["dtype"]]
    rows = lengths(case)
    total, brought = sum(n for n, _ in rows), sum(b for _, b in rows)
    kv = torch.randn(2, total, H, D, generator=g, device="cuda")
    kv[0] *= torch.exp(0.4 * torch.randn(H, D, generator=g, device="cuda"))      # some channels of keys are loud, and off zero
    kv[0] += 0.7 * torch.randn(H, D, generator=g, device="cuda")
    kv[1] *= 0.5
    q = torch.randn(brought, case["heads"], D, generator=g, device="cuda").to(t) if "heads" in case else None
    return kv.to(t), q, g


def prepare(case, seed):
    if case["kind"] == "copy":
        g = torch.Generator("cuda").manual_seed(seed * 7919 + 17)
        n = case["pages"] + 1
        pool = torch.randint(-2 ** 31, 2 ** 31 - 1, (case["layers"], n, page_bytes(case) // 4), generator=g, device="cuda", dtype=torch.int32)
        at = 1 + torch.randperm(n - 1, generator=g, device="cuda").to(torch.int32)
        return dict(case=case, pool=pool, src=at[:case["moved"]].clone(), dst=at[-case["moved"]:].clone())
    kv, q, g = rows_of(case, seed)
    rows, H, D, B = lengths(case), case["kv_heads"], case["dim"], case["seqs"]
    blocks = -(-max(n for n, _ in rows) // PAGE) + 1
    total = torch.tensor([n for n, _ in rows], dtype=torch.int32, device="cuda")
    brought = torch.tensor([b for _, b in rows], dtype=torch.int32, device="cuda")
    have = -(-total // PAGE)
    pages = int(have.sum()) + 1
    # every row's pages, scattered over the pool
    table = torch.zeros(B, blocks, dtype=torch.int32, device="cuda")
    held = torch.arange(blocks, device="cuda")[None] < have[:, None]
    table[held] = 1 + torch.randperm(pages - 1, generator=g, device="cuda").to(torch.int32)
    # the tokens that are there before the call, in their pages
    row = torch.repeat_interleave(torch.arange(B, device="cuda"), total.long())
    first = torch.cumsum(total.long(), 0) - total
    place = torch.arange(len(row), device="cuda") - first[row]
    new = place >= (total - brought)[row]
    slot = table[row, place // PAGE].long() * PAGE + place % PAGE
    fresh = case["kind"] == "append" or case["fresh"]
    old = ~new if fresh else torch.ones_like(new)
    codes = torch.zeros(2, pages * PAGE, H, D, dtype=torch.uint8, device="cuda")
    lo = torch.full((2, pages * PAGE, H, D // 64), math.nan, device="cuda")      # what no token has filled may hold anything
    step = torch.zeros(2, pages * PAGE, H, D // 64, device="cuda")
    codes[:, slot[old]], lo[:, slot[old]], step[:, slot[old]] = quantise(kv[:, old])
    pool = pages_of(codes.unflatten(1, (pages, PAGE)), lo.unflatten(1, (pages, PAGE)), step.unflatten(1, (pages, PAGE)), D)
    state = dict(case=case, pool=pool.reshape(1, pages, -1).contiguous(), table=table, start=total - brought, count=max(b for _, b in rows), keys=max(n for n, _ in rows))
    state["offsets"] = torch.cat([brought.new_zeros(1), torch.cumsum(brought, 0).to(torch.int32)])
    if fresh:
        state["k"], state["v"] = kv[0, new].contiguous(), kv[1, new].contiguous()
    if q is not None:
        state["q"] = q
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        from tinygpt_amd import ops
        if case["kind"] == "copy":
            ops.copy_pages(state["pool"], state["src"], state["dst"])
            return state["pool"]
        cache = ops.Kv4Cache(state["pool"], state["table"], case["kv_heads"], case["dim"])
        batch = dict(offsets=state["offsets"] if case["count"] > 1 else None, max_count=state["count"])
        if case["kind"] == "append":
            ops.kv4_append(cache, state["k"], state["v"], state["start"], **batch)
            return ops.kv4_read(cache, state["start"], len(state["k"]), dtype=state["k"].dtype, **batch)
        new = dict(k=state["k"], v=state["v"]) if case["fresh"] else {}
        out = ops.kv4_attend(cache, state["q"], state["start"], state["keys"], window=case["window"], **batch, **new)
        return (out, *ops.kv4_read(cache, state["start"], len(state["k"]), dtype=state["k"].dtype, **batch)) if case["fresh"] else out
    if case["kind"] == "copy":
        state["pool"][:, state["dst"].long()] = state["pool"][:, state["src"].long()]
        return state["pool"]
    kept = plain_append(state) if "k" in state else ()
    return kept if case["kind"] == "append" else (plain_attend(state), *kept) if kept else plain_attend(state)


def places(state):
    """row and place of every token that the call brings"""
    n = (state["offsets"][1:] - state["offsets"][:-1]).long()
    row = torch.repeat_interleave(torch.arange(len(n), device="cuda"), n, output_size=len(state["k"] if "k" in state else state["q"]))
    index = torch.arange(len(row), device="cuda") - state["offsets"].long()[row]
    return row, index, state["start"].long()[row] + index


def plain_append(state):
    """the tokens' codes and parameters into their pages; returns the values that the pages hold for them"""
    D, H = state["case"]["dim"], state["case"]["kv_heads"]
    row, _, place = places(state)
    n = (state["count"] + PAGE - 2) // PAGE + 1
    block = (state["start"].long() // PAGE)[:, None] + torch.arange(n, device="cuda")
    touched = torch.where(block < state["table"].shape[1], state["table"].gather(1, block.clamp(max=state["table"].shape[1] - 1)), 0).long()
    pool = state["pool"][0].view(-1, H, 4, 9 * D)
    codes, lo, step = (x.flatten(1, 3).contiguous() for x in parts_of(pool[touched], D))
    at = (row * n + place // PAGE - block[row, 0]) * PAGE + place % PAGE
    codes[:, at], lo[:, at], step[:, at] = quantise(torch.stack([state["k"], state["v"]]))
    held = value_of(codes[:, at], lo[:, at], step[:, at]).to(state["k"].dtype)
    pool[touched.flatten()] = pages_of(*(x.unflatten(1, (-1, PAGE)) for x in (codes, lo, step)), D)
    return held[0], held[1]


def plain_attend(state):
    case, q = state["case"], state["q"]
    D, H, B = case["dim"], case["kv_heads"], case["seqs"]
    row, index, place = places(state)
    C = state["count"]
    qs = torch.zeros(B, C, H, case["heads"] // H, D, device="cuda")
    qs[row, index] = q.float().unflatten(1, (H, -1))
    pos = torch.full((B, C), -1, dtype=torch.long, device="cuda")
    pos[row, index] = place
    words = state["pool"][0].view(-1, H, 4, 9 * D)[state["table"][:, :-(-state["keys"] // PAGE)].long()]
    codes, lo, step = parts_of(words, D)
    k, v = value_of(codes, lo, step).flatten(2, 3).transpose(2, 3)      # [rows][kv_heads][tokens][dim]
    del codes, words
    qs = qs.permute(0, 2, 3, 1, 4).flatten(2, 3) * D ** -0.5
    s = (qs @ k.transpose(-1, -2)).unflatten(2, (-1, C))                # [rows][kv_heads][heads of one][tokens brought][tokens]
    j = torch.arange(s.shape[-1], device="cuda")
    seen = j <= pos[..., None]
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    seen = seen[:, None, None]
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    p = (p / p.sum(-1, keepdim=True).clamp(min=1e-38)).flatten(2, 3)
    v = v.masked_fill(~seen.any(3)[:, 0].any(1)[:, None, :, None], 0.0)      # what no token sees may hold anything
    o = (p @ v).unflatten(2, (-1, C)).permute(0, 3, 1, 2, 4)
    return o[row, index].flatten(1, 2).to(q.dtype)


# ---- in 64 bits ---------------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "copy":
        return None
    kv, q, _ = rows_of(case, seed)
    held = []
    for x in kv:      # the levels that the format gives, their values in 64 bits
        codes, lo, step = quantise(x)
        held.append(value_of(codes.double(), lo.double(), step.double()))
    k, v = held
    rows, end, at, out, new = lengths(case), 0, 0, [], []
    for n, b in rows:
        end += n
        new.append(slice(end - b, end))
        if q is None:
            continue
        for c in range(0, b, 512):
            pos = n - b + c + torch.arange(min(512, b - c), device="cuda")
            qs = q[at + c:at + c + len(pos)].double().unflatten(1, (case["kv_heads"], -1))
            s = torch.einsum("chgd,thd->hgct", qs, k[end - n:end]) / math.sqrt(case["dim"])
            back = pos[:, None] - torch.arange(n, device="cuda")
            s[..., (back < 0) | (back >= (case["window"] or n + 1))] = -math.inf
            out.append(torch.einsum("hgct,thd->chgd", torch.softmax(s, -1), v[end - n:end]).flatten(1, 2))
        at += b
    kept = [torch.cat([x[s] for s in new]) for x in (k, v)]
    if q is None:
        return tuple(kept)
    return (torch.cat(out), *kept) if case["fresh"] else torch.cat(out)


def work(case):
    if case["kind"] == "copy":
        return {"bytes": 2 * case["moved"] * case["layers"] * page_bytes(case) + 8 * case["moved"], "flops": 0}
    H, D, es = case["kv_heads"], case["dim"], 4 if case["dtype"] == "fp32" else 2
    a_token = H * D * 9 // 8      # keys and values of one token, all heads, in the cache
    rows = lengths(case)
    brought = sum(b for _, b in rows)
    appended = brought * (4 * es * H * D + a_token) if case["kind"] == "append" or case["fresh"] else 0      # read, kept, given back
    if case["kind"] == "append":
        return {"bytes": appended, "flops": 0}
    bytes_, pairs = appended + 2 * brought * case["heads"] * D * es, 0
    for n, b in rows:
        w = case["window"] or n
        bytes_ += min(n, w + b - 1) * a_token
        pairs += sum(min(p + 1, w) for p in range(n - b, n))
    return {"bytes": bytes_, "flops": 4 * pairs * case["heads"] * D}
