"""Operators on tensors that a program holds itself: a key / value cache in 4 bits (append, read, attention over it) and page copies.

The same kernels serve a model whose option "kv.bits" is 4 (tinygpt_amd.ffi.Model); here the caller keeps the pages, the table and the positions, as torch tensors
on a GPU.  Format, page layout and what happens to pages that a table does not name: include/tgx.h, tgx_kv4_cache.  The reference's cache is a tensor per layer
that grows by concatenation (src/engine/CacheManager.h:24-51) and its attention is one library call over it (src/layer/Attention.h:103-112).

Every call runs on the current stream of the tensors' device and may be captured into a graph: positions, sequences and offsets are read on the device when
the call runs.  Tensors need no particular strides, only a head's channels lie together.  There are no gradients: tensors that ask
for one are refused.

torch brings a HIP runtime of its own, which the library shares if torch was loaded first: a program that uses both imports torch, or this module, before its first Model.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
import threading

import torch

from .ffi import TgxError, product_backend

PAGE_TOKENS = 128
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

# A call's structs (include/tgx.h) are packed into one buffer of the calling thread, at fixed places, and go to the library as addresses: a few calls of a step are short
# enough for their binding to count (an attention call: 22 us with a ctypes object a struct, 8 so, of which the library and its launches take half).
_CACHE, _BATCH, _ROWS = struct.Struct("QqQ5i4x"), struct.Struct("2iq3Q"), struct.Struct("Qi4x2q")
_AT_CACHE, _AT_BATCH, _AT_Q, _AT_K, _AT_V, _AT_OUT = 0, 64, 128, 160, 192, 224
_local = threading.local()


def _one_runtime(maps):
    """refuses a process (its memory map's lines) that holds two HIP runtimes: neither knows the other's memory and streams"""
    found = sorted({line.split()[-1] for line in maps if "/libamdhip64.so" in line})
    if len(found) > 1:
        raise RuntimeError(f"two HIP runtimes are loaded ({', '.join(found)}): import torch or tinygpt_amd.ops before the first Model of the process")


class _Calls:
    """the library's entry points, addresses as integers"""

    def __init__(self):
        self.be = product_backend()
        with open("/proc/self/maps") as maps:
            _one_runtime(maps)
        p, i, q, f = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
        for name, res, args in (("kv4_append", i, [p] * 4 + [i, p]), ("kv4_read", i, [p] * 4 + [i, p]), ("kv4_attend_workspace", q, [p, p, i, i, q, i]),
                                ("kv4_attend", i, [p, p, p, i, p, p, f, i, q, p, p, q, i, p]), ("copy_pages", i, [p, q, q, p, q, q, i, q, p, p, i, i, p])):
            setattr(self, name, ctypes.CFUNCTYPE(res, *args)(ctypes.cast(getattr(self.be.lib, "tgx_" + name), ctypes.c_void_p).value))

    def check(self, status):
        if status:
            raise TgxError(status, (self.be.op_last_error() or b"").decode())


@functools.lru_cache(maxsize=None)
def _calls() -> _Calls:
    return _Calls()


def _buffer():
    try:
        return _local.buf, _local.at
    except AttributeError:
        _local.buf = ctypes.create_string_buffer(256)
        _local.at = ctypes.addressof(_local.buf)
        return _local.buf, _local.at


@functools.lru_cache(maxsize=1024)
def _workspace(entries, max_count, tokens, kv_heads, head_dim, heads, window, max_keys, device):
    """bytes of an attention call's workspace: a function of sizes"""
    cache, batch = _CACHE.pack(16, 1, 16, 1, 1, 1, kv_heads, head_dim), _BATCH.pack(entries, max_count, tokens, 0, 16, 0 if tokens == entries and max_count == 1 else 16)
    return max(0, _calls().kv4_attend_workspace(ctypes.cast(cache, ctypes.c_void_p), ctypes.cast(batch, ctypes.c_void_p), heads, window, max_keys, device))


def _whole_pages(max_keys):
    """the keys by which work is divided: pages of them count, so that a row's workspace is looked up anew once a page and not with every token"""
    return min(-(-max_keys // PAGE_TOKENS) * PAGE_TOKENS, 2 ** 31 - 1)


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
        if head_dim not in (64, 128) or kv_heads < 1:
            raise ValueError(f"a 4-bit cache of {kv_heads} heads of {head_dim} channels is not built (head_dim 64 and 128 are)")
        nbytes, shape, device = kv_heads * head_dim * 144, pool.shape, pool.device
        if len(shape) < 3 or not pool.is_contiguous() or math.prod(shape[2:]) * pool.element_size() != nbytes:
            raise ValueError(f"pool: contiguous [layers][pages][...] with {nbytes} bytes a page")
        if table.dtype is not torch.int32 or table.dim() != 2:
            raise ValueError("table: int32 [sequences][pages of one]")
        (seqs, length), (stride, one) = table.shape, table.stride()
        if length > 1 and one != 1 or seqs > 1 and stride < length:
            raise ValueError("table: a sequence's entries lie together and are its own")
        if device.type != "cuda" or device != table.device:
            raise ValueError(f"pool ({device}) and table ({table.device}) are on one GPU")
        self.pool, self.table, self.kv_heads, self.head_dim, self.device, self.index, self.layers = pool, table, kv_heads, head_dim, device, device.index, shape[0]
        self._at, self._layer_bytes = pool.data_ptr(), shape[1] * nbytes
        self._rest = (shape[1], table.data_ptr(), stride if seqs > 1 else length, length, seqs, kv_heads, head_dim)

    @classmethod
    def empty(cls, layers: int, pages: int, kv_heads: int, head_dim: int, seqs: int, max_tokens: int, device="cuda"):
        """a pool of `pages` pages a layer and a table whose entries name no page"""
        pool = torch.empty(layers, pages, kv4_page_bytes(kv_heads, head_dim), dtype=torch.uint8, device=device)
        return cls(pool, torch.full((seqs, -(-max_tokens // PAGE_TOKENS)), -1, dtype=torch.int32, device=device), kv_heads, head_dim)

    def _pack(self, buf, layer):
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        _CACHE.pack_into(buf, _AT_CACHE, self._at + layer * self._layer_bytes, *self._rest)


def _int32(name, t, n, device):
    if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name}: int32 [{n}] without gaps on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _pack_batch(buf, cache, tokens, start, seq, offsets, max_count):
    """(entries, max_count)"""
    entries, dev = len(start) if start.dim() == 1 else -1, cache.device
    if offsets is None:
        if tokens != entries:
            raise ValueError(f"{tokens} tokens of {entries} entries without offsets (an entry brings one)")
        max_count = 1
    elif max_count is None:
        max_count = tokens
    _BATCH.pack_into(buf, _AT_BATCH, entries, max_count, tokens, 0 if seq is None else _int32("seq", seq, entries, dev), _int32("start", start, entries, dev),
                     0 if offsets is None else _int32("offsets", offsets, entries + 1, dev))
    return entries, max_count


def _pack_rows(buf, at, name, t, tokens, heads, cache):
    if t.shape != (tokens, heads, cache.head_dim):
        raise ValueError(f"{name}: [{tokens}][{heads}][{cache.head_dim}], got {tuple(t.shape)}")
    dtype = _DTYPES.get(t.dtype)
    if dtype is None:
        raise ValueError(f"{name}: bfloat16, float16 or float32, got {t.dtype}")
    if t.device != cache.device:
        raise ValueError(f"{name} is on {t.device}, the cache on {cache.device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and a 4-bit cache has none: torch.no_grad() or detach()")
    token, head, channel = t.stride()
    if channel != 1:
        raise ValueError(f"{name}: a head's channels lie together (stride 1)")
    _ROWS.pack_into(buf, at, t.data_ptr(), dtype, token, head)


_stream = torch._C._cuda_getCurrentRawStream      # of a device's index; as torch.cuda.current_stream(device).cuda_stream, without the object around it (0.1 us for 1.9)


def kv4_append(cache: Kv4Cache, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, layer: int = 0, seq: torch.Tensor = None, offsets: torch.Tensor = None,
               max_count: int = None):
    """Keys and values [tokens][kv_heads][head_dim] into the cache's pages (== KVCacheManager::append).

    Entry e brings tokens offsets[e] .. offsets[e + 1] - 1 (int32 [entries + 1]; None: the one token e) of sequence seq[e] (None: e), at positions start[e], start[e] +
    1, ...  max_count: the most that an entry brings (None: all tokens; a smaller grid where it is given).  Positions behind the table's pages are left out."""
    c, (buf, at) = _calls(), _buffer()
    tokens = len(k)
    _pack_batch(buf, cache, tokens, start, seq, offsets, max_count)
    _pack_rows(buf, _AT_K, "k", k, tokens, cache.kv_heads, cache)
    _pack_rows(buf, _AT_V, "v", v, tokens, cache.kv_heads, cache)
    cache._pack(buf, layer)
    c.check(c.kv4_append(at + _AT_CACHE, at + _AT_BATCH, at + _AT_K, at + _AT_V, cache.index, _stream(cache.index)))


def kv4_read(cache: Kv4Cache, start: torch.Tensor, tokens: int, dtype: torch.dtype = torch.float32, layer: int = 0, seq: torch.Tensor = None, offsets: torch.Tensor = None,
             max_count: int = None, out=None):
    """The values that the cache holds for a batch's tokens, named as in kv4_append: (keys, values), each [tokens][kv_heads][head_dim], rounded once to dtype.
    out: tensors to write to; tokens that no entry names or that have a negative position stay as they were in them (in new ones they hold anything), tokens without a page read as zeros."""
    c, (buf, at) = _calls(), _buffer()
    k, v = out if out is not None else torch.empty((2, tokens, cache.kv_heads, cache.head_dim), dtype=dtype, device=cache.device).unbind(0)
    _pack_batch(buf, cache, tokens, start, seq, offsets, max_count)
    _pack_rows(buf, _AT_K, "k", k, tokens, cache.kv_heads, cache)
    _pack_rows(buf, _AT_V, "v", v, tokens, cache.kv_heads, cache)
    cache._pack(buf, layer)
    c.check(c.kv4_read(at + _AT_CACHE, at + _AT_BATCH, at + _AT_K, at + _AT_V, cache.index, _stream(cache.index)))
    return k, v


def kv4_attend(cache: Kv4Cache, q: torch.Tensor, start: torch.Tensor, max_keys: int, layer: int = 0, seq: torch.Tensor = None, offsets: torch.Tensor = None,
               max_count: int = None, scale: float = None, window: int = 0, k: torch.Tensor = None, v: torch.Tensor = None, out: torch.Tensor = None) -> torch.Tensor:
    """Attention of queries [tokens][heads][head_dim] over the cache (== flashAttention over what the reference's cache returns).

    The batch's tokens are named as in kv4_append; a token at position p sees its sequence's keys at 0 .. p, with window > 0 the last `window` of them.  k, v: the tokens'
    own keys and values, which join the cache first (a token sees itself, and what other entries bring in front of it in its sequence); without them they are there already.  max_keys: at least the last position + 1 of every
    entry.  max_keys and max_count (the most that an entry brings; None: all tokens) choose the kernel and divide the work, for all entries alike: name the count where it is known, and attend for
    single tokens of long rows in a call of their own, not in one with portions.  scale: head_dim ** -0.5 where not given.  A token that sees nothing gets zeros; one that no entry names stays as it was in `out` (in a
    new one it holds anything)."""
    c, (buf, at) = _calls(), _buffer()
    if q.dim() != 3:
        raise ValueError(f"q: [tokens][heads][{cache.head_dim}], got {tuple(q.shape)}")
    tokens, heads, _ = q.shape
    entries, max_count = _pack_batch(buf, cache, tokens, start, seq, offsets, max_count)
    _pack_rows(buf, _AT_Q, "q", q, tokens, heads, cache)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.dtype != q.dtype:
        raise ValueError(f"out: {q.dtype} as q, got {out.dtype}")
    _pack_rows(buf, _AT_OUT, "out", out, tokens, heads, cache)
    if (k is None) != (v is None):
        raise ValueError("k and v come together")
    if k is not None:
        _pack_rows(buf, _AT_K, "k", k, tokens, cache.kv_heads, cache)
        _pack_rows(buf, _AT_V, "v", v, tokens, cache.kv_heads, cache)
    cache._pack(buf, layer)
    index = cache.index
    need = _workspace(entries, max_count, tokens, cache.kv_heads, cache.head_dim, heads, window, _whole_pages(max_keys), index)
    ws = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
    c.check(c.kv4_attend(at + _AT_CACHE, at + _AT_BATCH, at + _AT_Q, heads, None if k is None else at + _AT_K, None if k is None else at + _AT_V, cache.head_dim ** -0.5 if scale is None else scale,
                         window, max_keys, at + _AT_OUT, ws.data_ptr() if need else None, need, index, _stream(index)))
    return out


def copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, into: torch.Tensor = None):
    """Pages between the layers' pools of paged caches, 4-bit or 16-bit: page dst[i] of `into` (None: of pool itself) becomes page src[i] of pool, in every layer.

    pool, into: [layers][pages][...] whose pages lie without gaps, a multiple of 16 bytes each; src, dst: int32.  A pair with a page that does not exist is left out;
    a page that is copied from is not copied to in the same call, and none is copied to twice."""
    n = len(src) if src.dim() == 1 else -1
    sizes = []
    for name, t in (("pool", pool),) if into is None else (("pool", pool), ("into", into)):
        shape = t.shape
        if len(shape) < 3 or not t.is_cuda or not t.is_contiguous() and t.numel() and not t[0].is_contiguous():
            raise ValueError(f"{name}: [layers][pages][...] on a GPU, a layer's pages without gaps")
        es = t.element_size()
        sizes.append((t.data_ptr(), shape[1], t.stride(0) * es, shape[0], shape[2:].numel() * es))
    a, b = sizes[0], sizes[-1]
    if into is not None and (a[3:] != b[3:] or pool.device != into.device):
        raise ValueError(f"pools of {a[3]} and {b[3]} layers, pages of {a[4]} and {b[4]} bytes, on {pool.device} and {into.device}")
    dev = pool.device
    c = _calls()
    c.check(c.copy_pages(*a[:3], *b[:3], a[3], a[4], _int32("src", src, n, dev), _int32("dst", dst, n, dev), n, dev.index, _stream(dev.index)))
    return pool if into is None else into
