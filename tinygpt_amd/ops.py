"""Operators on tensors that a program holds itself: a key / value cache in 4 bits (append, read, attention over it) and page copies.

The same kernels serve a model whose option "kv.bits" is 4 (tinygpt_amd.ffi.Model); here the caller keeps the pages, the table and the positions, as torch tensors
on a GPU.  Format, page layout and what happens to pages that a table does not name: include/tgx.h, tgx_kv4_cache.  The reference's cache is a tensor per layer
that grows by concatenation (src/engine/CacheManager.h:24-51) and its attention is one library call over it (src/layer/Attention.h:103-112).

Every call runs on the current stream of the tensors' device and may be captured into a graph: positions, sequences and offsets are read on the device when
the call runs.  Tensors need no particular strides, only a head's channels lie together.
"""
from __future__ import annotations

import ctypes

import torch

from .ffi import Kv4BatchArg, Kv4CacheArg, Kv4RowsArg, TgxError, product_backend

PAGE_TOKENS = 128
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def kv4_page_bytes(kv_heads: int, head_dim: int) -> int:
    """bytes of a page (128 tokens of all key / value heads of a layer)"""
    n = product_backend().kv4_page_bytes(kv_heads, head_dim)
    if n < 0:
        raise ValueError(f"a 4-bit cache of {kv_heads} heads of {head_dim} channels is not built (head_dim 64 and 128 are)")
    return n


class Kv4Cache:
    """Pages and page table of a 4-bit cache.

    pool: contiguous [layers][pages][...] of any type, kv4_page_bytes(kv_heads, head_dim) bytes a page; table: int32 [sequences][pages of one], the pages of a
    sequence's tokens 0-127, 128-255, ...  Both stay the caller's: pages are assigned by writing the table.  What a page holds where nothing was appended
    does not matter."""

    def __init__(self, pool: torch.Tensor, table: torch.Tensor, kv_heads: int, head_dim: int):
        nbytes = kv_heads * head_dim * 144
        if head_dim not in (64, 128) or kv_heads < 1:
            raise ValueError(f"a 4-bit cache of {kv_heads} heads of {head_dim} channels is not built (head_dim 64 and 128 are)")
        if pool.dim() < 3 or not pool.is_contiguous() or pool[0, 0].numel() * pool.element_size() != nbytes if pool.numel() else pool.dim() < 3:
            raise ValueError(f"pool: contiguous [layers][pages][...] with {nbytes} bytes a page")
        if table.dtype != torch.int32 or table.dim() != 2 or table.stride(1) != 1 and table.shape[1] > 1:
            raise ValueError("table: int32 [sequences][pages of one], a sequence's entries together")
        if not pool.is_cuda or pool.device != table.device:
            raise ValueError(f"pool ({pool.device}) and table ({table.device}) are on one GPU")
        self.pool, self.table, self.kv_heads, self.head_dim = pool, table, kv_heads, head_dim
        self.device = pool.device
        self._rows_of = {kv_heads: (kv_heads, head_dim)}
        self._layer_bytes = pool.shape[1] * nbytes
        stride = table.stride(0) if table.shape[0] > 1 else table.shape[1]
        if stride < table.shape[1]:
            raise ValueError("table: a sequence's entries are its own")
        self._arg = Kv4CacheArg(pool.data_ptr(), pool.shape[1], table.data_ptr(), stride, table.shape[1], table.shape[0], kv_heads, head_dim)

    @classmethod
    def empty(cls, layers: int, pages: int, kv_heads: int, head_dim: int, seqs: int, max_tokens: int, device="cuda"):
        """a pool of `pages` pages a layer and a table whose entries name no page"""
        pool = torch.empty(layers, pages, kv4_page_bytes(kv_heads, head_dim), dtype=torch.uint8, device=device)
        return cls(pool, torch.full((seqs, -(-max_tokens // PAGE_TOKENS)), -1, dtype=torch.int32, device=device), kv_heads, head_dim)

    def _at(self, layer: int) -> Kv4CacheArg:
        if not 0 <= layer < self.pool.shape[0]:
            raise ValueError(f"layer {layer} of {self.pool.shape[0]}")
        self._arg.pool = self.pool.data_ptr() + layer * self._layer_bytes
        return self._arg


def _int32(name, t, n, device):
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or t.stride(0) != 1 and n > 1 or t.device != device:
        raise ValueError(f"{name}: int32 [{n}] without gaps on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _batch(cache, tokens, start, seq, offsets, max_count):
    entries, dev = start.shape[0], cache.device
    if offsets is None:
        if tokens != entries:
            raise ValueError(f"{tokens} tokens of {entries} entries without offsets (an entry brings one)")
        max_count = 1
    elif max_count is None:
        max_count = tokens
    return Kv4BatchArg(entries, max_count, tokens, None if seq is None else _int32("seq", seq, entries, dev), _int32("start", start, entries, dev),
                       None if offsets is None else _int32("offsets", offsets, entries + 1, dev))


def _rows(name, t, heads, cache):
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != cache.head_dim:
        raise ValueError(f"{name}: [tokens][{heads}][{cache.head_dim}], got {tuple(t.shape)}")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name}: bfloat16, float16 or float32, got {t.dtype}")
    if t.device != cache.device:
        raise ValueError(f"{name} is on {t.device}, the cache on {cache.device}")
    if t.stride(2) != 1:
        raise ValueError(f"{name}: a head's channels lie together (stride 1)")
    return Kv4RowsArg(t.data_ptr(), _DTYPES[t.dtype], t.stride(0), t.stride(1))


def _check(be, status):
    if status:
        raise TgxError(status, (be.op_last_error() or b"").decode())


def _where(device):
    return device.index, torch.cuda.current_stream(device).cuda_stream


def kv4_append(cache: Kv4Cache, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, layer: int = 0, seq: torch.Tensor = None, offsets: torch.Tensor = None,
               max_count: int = None):
    """Keys and values [tokens][kv_heads][head_dim] into the cache's pages (== KVCacheManager::append).

    Entry e brings tokens offsets[e] .. offsets[e + 1] - 1 (int32 [entries + 1]; None: the one token e) of sequence seq[e] (None: e), at positions start[e], start[e] +
    1, ...  max_count: the most that an entry brings (None: all tokens; a smaller grid where it is given).  Positions behind the table's pages are left out."""
    be = product_backend()
    b = _batch(cache, k.shape[0], start, seq, offsets, max_count)
    ka, va = _rows("k", k, cache.kv_heads, cache), _rows("v", v, cache.kv_heads, cache)
    if v.shape[0] != k.shape[0]:
        raise ValueError(f"{k.shape[0]} keys and {v.shape[0]} values")
    _check(be, be.kv4_append(cache._at(layer), b, ka, va, *_where(cache.device)))


def kv4_read(cache: Kv4Cache, start: torch.Tensor, tokens: int, dtype: torch.dtype = torch.float32, layer: int = 0, seq: torch.Tensor = None, offsets: torch.Tensor = None,
             max_count: int = None, out=None):
    """The values that the cache holds for a batch's tokens, named as in kv4_append: (keys, values), each [tokens][kv_heads][head_dim], rounded once to dtype.
    out: tensors to write to; tokens that no entry names stay as they were in them."""
    be = product_backend()
    k, v = out if out is not None else torch.empty(2, tokens, cache.kv_heads, cache.head_dim, dtype=dtype, device=cache.device)
    if k.shape[0] != tokens or v.shape[0] != tokens:
        raise ValueError(f"out: {tokens} tokens each")
    b = _batch(cache, tokens, start, seq, offsets, max_count)
    _check(be, be.kv4_read(cache._at(layer), b, _rows("k", k, cache.kv_heads, cache), _rows("v", v, cache.kv_heads, cache), *_where(cache.device)))
    return k, v


def kv4_attend(cache: Kv4Cache, q: torch.Tensor, start: torch.Tensor, max_keys: int, layer: int = 0, seq: torch.Tensor = None, offsets: torch.Tensor = None,
               max_count: int = None, scale: float = None, window: int = 0, k: torch.Tensor = None, v: torch.Tensor = None, out: torch.Tensor = None) -> torch.Tensor:
    """Attention of queries [tokens][heads][head_dim] over the cache (== flashAttention over what the reference's cache returns).

    The batch's tokens are named as in kv4_append; a token at position p sees its sequence's keys at 0 .. p, with window > 0 the last `window` of them.  k, v: the tokens'
    own keys and values, which join the cache first (then a token sees itself); without them they are there already.  max_keys: at least the last position + 1 of every
    entry, to divide the work by.  scale: head_dim ** -0.5 where not given.  A token that sees nothing gets zeros."""
    be = product_backend()
    heads = q.shape[1] if q.dim() == 3 else 0
    b = _batch(cache, q.shape[0], start, seq, offsets, max_count)
    qa = _rows("q", q, heads, cache)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out: as q")
    oa = _rows("out", out, heads, cache)
    ka = va = None
    if (k is None) != (v is None):
        raise ValueError("k and v come together")
    if k is not None:
        if k.shape[0] != q.shape[0] or v.shape[0] != q.shape[0]:
            raise ValueError(f"{q.shape[0]} queries, {k.shape[0]} keys and {v.shape[0]} values")
        ka, va = _rows("k", k, cache.kv_heads, cache), _rows("v", v, cache.kv_heads, cache)
    c = cache._at(layer)
    device, stream = _where(cache.device)
    need = be.kv4_attend_workspace(c, b, heads, window, max_keys, device)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    _check(be, be.kv4_attend(c, b, qa, heads, ka, va, cache.head_dim ** -0.5 if scale is None else scale, window, max_keys, oa, None if ws is None else ws.data_ptr(), max(need, 0),
                             device, stream))
    return out


def copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, into: torch.Tensor = None):
    """Pages between the layers' pools of paged caches, 4-bit or 16-bit: page dst[i] of `into` (None: of pool itself) becomes page src[i] of pool, in every layer.

    pool, into: [layers][pages][...] whose pages lie without gaps, a multiple of 16 bytes each; src, dst: int32.  A pair with a page that does not exist is left out;
    a page that is copied from is not copied to in the same call, and none is copied to twice."""
    into = pool if into is None else into
    be = product_backend()
    sizes = []
    for name, t in (("pool", pool), ("into", into)):
        if t.dim() < 3 or not t.is_cuda or t.numel() and not t[0].is_contiguous():
            raise ValueError(f"{name}: [layers][pages][...] on a GPU, a layer's pages without gaps")
        sizes.append(t.shape[2:].numel() * t.element_size())
    if sizes[0] != sizes[1] or pool.shape[0] != into.shape[0] or pool.device != into.device:
        raise ValueError(f"pools of {pool.shape[0]} and {into.shape[0]} layers, pages of {sizes[0]} and {sizes[1]} bytes, on {pool.device} and {into.device}")
    n = src.shape[0] if src.dim() == 1 else -1
    args = (_int32("src", src, n, pool.device), _int32("dst", dst, n, pool.device), n)
    _check(be, be.copy_pages(pool.data_ptr(), pool.shape[1], pool.stride(0) * pool.element_size(), into.data_ptr(), into.shape[1], into.stride(0) * into.element_size(),
                             pool.shape[0], sizes[0], *args, *_where(pool.device)))
    return into
