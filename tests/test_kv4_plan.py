"""The 4-bit cache's arithmetic on sizes (tinygpt_amd/csrc/kv4_plan.h), compiled with the host compiler: where codes lie, what entries and pages out of range come to, how the
keys are divided; and what the operators refuse before anything reaches a GPU."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT

SOURCE = r"""
#include "kv4_plan.h"
#include <cstring>
#include <vector>
using namespace tgx;
// 0: every code of a block has a place of its own inside its part, every parameter a word
extern "C" int places(int hd) {
  std::vector<unsigned> w(9 * hd, 0u);
  for (int t = 0; t < 32; t++)
    for (int c = 0; c < hd; c++) {
      const int k = kv4_key_word(hd, t, c), v = kv4_value_word(hd, t, c);
      if (k < 0 || k >= 4 * hd || v < 4 * hd || v >= 8 * hd) return 1;
      const unsigned kb = 15u << kv4_key_bit(c), vb = 15u << kv4_value_bit(t);
      if ((w[k] & kb) || (w[v] & vb)) return 2;
      w[k] |= kb; w[v] |= vb;
      if (kv4_value_token((t & 15) >> 2, (t & 3) + 4 * (t >> 4)) != t) return 3;
    }
  for (int t = 0; t < 32; t++)
    for (int x = 0; x < 2; x++)
      for (int g = 0; g < hd / 64; g++) {
        const int p = kv4_param_word(hd, t, x, g);
        if (p < 8 * hd || p >= 9 * hd || w[p]) return 4;
        w[p] = ~0u;
      }
  for (unsigned x : w) if (x != ~0u) return 5;
  return 0;
}
// what an entry brings: count, or -1 - (first token) to tell that it is all outside
extern "C" int entry(int seqs, int seq, int start, int o0, int o1, long long tokens, int max_count) {
  int off[2] = {o0, o1};
  Kv4Args a{};
  a.seqs = seqs; a.seq = &seq; a.start = &start; a.offsets = off; a.tokens = tokens; a.max_count = max_count; a.entries = 1; a.each = 1;
  const Kv4Entry n = kv4_entry(a, 0);
  if (n.count && (n.seq < 0 || n.seq >= seqs || n.tok0 < 0 || n.tok0 + n.count > tokens || n.count > max_count || (long long)n.start + n.count > 0x7fffffffLL)) return -1;
  return n.count;
}
// a page's first word, -1: none
extern "C" long long page(int p, int pages, int b, int len, int kvh, int heads, int hd) {
  std::vector<int> t((size_t)len, p);
  static unsigned int base[1];
  Kv4Args a{};
  a.pool = base; a.pages = pages; a.table = t.data(); a.table_stride = len; a.table_len = len; a.seqs = 1; a.kv_heads = heads;
  const unsigned int* w = kv4_page(a, 0, b, kvh, hd);
  return w ? (long long)(((size_t)w - (size_t)base) / 4) : -1;
}
// 0: the splits hold every page that a column can see once and none twice
extern "C" int ranges(int first, int last, int window, int len, int splits) {
  int next = -1, end = 0;
  for (int s = 0; s < splits; s++) {
    const Kv4Range r = kv4_range(first, last, window, len, s, splits);
    if (r.lo > r.hi || r.lo < 0 || (r.hi > len && r.hi > r.lo)) return 1;
    if (r.lo == r.hi) continue;
    if (next >= 0 && r.lo != next) return 2;
    if (next < 0) { const int lo = window > 0 && first - window + 1 > 0 ? first - window + 1 : 0; if (r.lo != lo / 128) return 3; }
    next = end = r.hi;
  }
  const int want = last < 0 ? 0 : (last / 128 + 1 < len ? last / 128 + 1 : len), lo = window > 0 && first - window + 1 > 0 ? (first - window + 1) / 128 : 0;
  return end == (want > lo ? want : 0) ? 0 : 4;
}
extern "C" void plan(int entries, int max_count, int kv_heads, int group, int hd, int window, long long keys, int cus, int* out) {
  const Kv4Plan p = kv4_plan(entries, max_count, kv_heads, group, hd, window, keys, cus);
  out[0] = p.kw; out[1] = p.nt; out[2] = p.tiles; out[3] = p.splits;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv4")
    src, lib = d / "plan.cpp", d / "libplan.so"
    src.write_text(SOURCE)
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "tinygpt_amd", "csrc"), str(src), "-o", str(lib)])
    so = ctypes.CDLL(str(lib))
    so.page.restype = ctypes.c_longlong
    so.entry.argtypes = [ctypes.c_int] * 5 + [ctypes.c_longlong, ctypes.c_int]
    so.plan.argtypes = [ctypes.c_int] * 6 + [ctypes.c_longlong, ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    return so


@pytest.mark.parametrize("hd", [64, 128])
def test_every_code_has_a_place(plan, hd):
    assert plan.places(hd) == 0


def test_entries_out_of_range_bring_nothing(plan):
    assert plan.entry(4, 3, 100, 2, 7, 9, 16) == 5
    assert plan.entry(4, 3, 100, 2, 7, 9, 3) == 3                       # at most max_count
    assert plan.entry(4, 3, -7, 2, 7, 9, 16) == 5                       # a negative position is the kernels' own business
    big = 2 ** 31 - 1
    for seqs, seq, start, o0, o1, tokens, most in [(4, 4, 0, 0, 1, 1, 1), (4, -1, 0, 0, 1, 1, 1), (0, 0, 0, 0, 1, 1, 1), (4, 0, 0, -1, 1, 5, 9), (4, 0, 0, 3, 1, 5, 9),
                                                   (4, 0, 0, 3, 9, 5, 9), (4, 0, big, 0, 1, 5, 9), (4, 0, big - 3, 0, 5, 5, 9), (4, 0, 0, big, big, 5, 9), (4, 0, 0, -big - 1, big, 5, 9)]:
        assert plan.entry(seqs, seq, start, o0, o1, tokens, most) in (0, ), (seqs, seq, start, o0, o1)
    assert plan.entry(4, 0, -big - 1, 0, 5, 5, 9) == 5


def test_pages_out_of_range_are_none(plan):
    assert plan.page(6, 7, 2, 3, 1, 8, 128) == (6 * 8 + 1) * 36 * 128
    assert plan.page(40000, 70000, 0, 1, 7, 8, 128) == (40000 * 8 + 7) * 36 * 128      # beyond 32 bits
    for p, pages, b in [(-1, 7, 0), (7, 7, 0), (2 ** 31 - 1, 7, 0), (-2 ** 31, 7, 0), (0, 0, 0), (3, 7, -1), (3, 7, 3), (3, 7, 2 ** 24)]:
        assert plan.page(p, pages, b, 3, 0, 8, 64) == -1


def test_splits_hold_every_page_once(plan):
    for last in [-5, -1, 0, 1, 127, 128, 129, 1000, 5000]:
        for back in [0, 1, 5, 200]:
            for window in [0, 1, 2, 100, 128, 129, 4000]:
                for length in [0, 1, 2, 9, 50]:
                    for splits in [1, 2, 3, 7, 64]:
                        assert plan.ranges(last - back, last, window, length, splits) == 0, (last, back, window, length, splits)


@pytest.mark.parametrize("cus", [1, 64, 256])
def test_plans_cover_their_columns(plan, cus):
    out = (ctypes.c_int * 4)()
    for entries in [1, 3, 64, 65535]:
        for count in [1, 2, 5, 17, 200, 2048, 65535]:
            for group in [1, 4, 7, 16]:
                for window, keys in [(0, 1), (0, 131072), (64, 131072), (0, 2 ** 31 - 1), (0, 0)]:
                    for hd in (64, 128):
                        plan.plan(entries, count, 8, group, hd, window, keys, cus, out)
                        kw, nt, tiles, splits = out
                        assert kw in (1, 4, 8) and tiles * 16 * nt * (1 if kw > 1 else 4) >= count * group and 1 <= splits <= 256
                        assert kw < 8 or count == 1 and group <= 8
                        if kw > 1 and nt == 1:
                            assert tiles == 1      # a single token's keys and values are appended by one workgroup a (entry, head, split)


# ---- what is refused, before a GPU is touched ---------------------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def be():
    from tinygpt_amd import build
    from tinygpt_amd.ffi import Backend
    return Backend(build.build_lib(), "tgx_")


def call(be, name="append", pages=4, table_stride=3, table_len=3, seqs=2, kv_heads=2, head_dim=64, pool=4096, entries=2, max_count=1, tokens=2, offsets=None, start=4096, dtype=1,
         vdtype=1, data=4096, heads=4, window=0, keys=300, ws=4096, ws_bytes=1 << 40, scale=0.125, out=1, with_v=True):
    from tinygpt_amd.ffi import Kv4BatchArg, Kv4CacheArg, Kv4RowsArg
    c = Kv4CacheArg(pool, pages, 4096, table_stride, table_len, seqs, kv_heads, head_dim)
    b = Kv4BatchArg(entries, max_count, tokens, None, start, offsets)
    k, v = Kv4RowsArg(data, dtype, 128, 64), Kv4RowsArg(data, vdtype, 128, 64)
    if name == "attend":
        return be.kv4_attend(c, b, k, heads, k, v if with_v else None, scale, window, keys, Kv4RowsArg(data, out, 128, 64), ws, ws_bytes, 0, None)
    return getattr(be, "kv4_" + name)(c, b, k, v, 0, None)


INVALID, UNSUPPORTED = 1, 2
REFUSED = [("head_dim", 96, UNSUPPORTED), ("head_dim", 0, UNSUPPORTED), ("kv_heads", 0, INVALID), ("kv_heads", -3, INVALID), ("pages", -1, INVALID), ("seqs", -1, INVALID),
           ("table_len", 4, INVALID), ("table_len", -1, INVALID), ("entries", -1, INVALID), ("entries", 65536, INVALID), ("tokens", 3, INVALID), ("tokens", -1, INVALID), ("max_count", -1, INVALID),
           ("pool", 4100, INVALID), ("pool", None, INVALID), ("start", None, INVALID), ("dtype", 3, INVALID), ("vdtype", 2, INVALID), ("data", None, INVALID), ("data", 4097, INVALID)]


@pytest.mark.parametrize("name", ["append", "read", "attend"])
@pytest.mark.parametrize("key,value,status", REFUSED)
def test_refusals(be, name, key, value, status):
    assert call(be, name, **{key: value}) == status
    assert be.op_last_error()


@pytest.mark.parametrize("key,value,status", [("heads", 3, INVALID), ("heads", 0, INVALID), ("heads", -4, INVALID), ("heads", 34, UNSUPPORTED), ("window", -1, INVALID), ("window", 2 ** 30 + 1, INVALID),
                                              ("keys", -1, INVALID), ("keys", 2 ** 31, INVALID), ("scale", float("nan"), INVALID), ("scale", float("inf"), INVALID), ("out", 2, INVALID), ("with_v", False, INVALID)])
def test_attention_refusals(be, key, value, status):
    assert call(be, "attend", **{key: value}) == status
    assert be.op_last_error()


def test_nothing_to_do_needs_nothing(be):
    for name in ("append", "read", "attend"):
        assert call(be, name, entries=0, tokens=0, pool=None, start=None, data=None) == 0
    assert be.copy_pages(None, 0, 0, None, 0, 0, 3, 64, None, None, 0, 0, None) == 0


def test_page_copy_refusals(be):
    good = dict(src=4096, src_pages=4, src_stride=4096, dst=8192, dst_pages=4, dst_stride=4096, layers=2, page_bytes=256, frm=4096, to=4096, n=2, device=0, stream=None)
    for key, value in [("n", -1), ("n", 65536), ("layers", -1), ("page_bytes", 24), ("page_bytes", -16), ("src_stride", 8), ("dst_stride", -16), ("src", None), ("dst", 8196), ("frm", None), ("to", None),
                       ("src_pages", -1), ("dst_pages", -1)]:
        assert be.copy_pages(*dict(good, **{key: value}).values()) == INVALID, key


def test_page_bytes(be):
    assert be.kv4_page_bytes(8, 128) == 8 * 128 * 144 and be.kv4_page_bytes(2, 64) == 2 * 64 * 144
    assert be.kv4_page_bytes(8, 96) == -1 and be.kv4_page_bytes(0, 64) == -1


def test_tensors_are_checked_before_the_library():
    """the refusals of tinygpt_amd.ops that tensors on a CPU show"""
    import torch
    from tinygpt_amd import ops
    pool, table = torch.zeros(1, 2, 2 * 64 * 144, dtype=torch.uint8), torch.zeros(2, 3, dtype=torch.int32)
    for args in [(pool, table, 2, 96), (pool, table, 0, 64), (pool, table, 4, 64), (pool[0], table, 2, 64), (pool, table.long(), 2, 64), (pool, table[0], 2, 64), (pool, table, 2, 64)]:
        with pytest.raises(ValueError):
            ops.Kv4Cache(*args)      # the last: not on a GPU
    for args in [(pool, table[0], table[0]), (pool[0], table[0], table[0])]:
        with pytest.raises(ValueError):
            ops.copy_pages(*args)


def test_two_runtimes_are_refused():
    from tinygpt_amd import ops
    line = "7f0000000000-7f0000001000 r-xp 00000000 08:01 42    {}\n".format
    one = [line("/opt/rocm/lib/libamdhip64.so.7"), line("/opt/rocm/lib/libamdhip64.so.7"), line("/lib/libc.so.6"), "7f00-7f10 rw-p 0 00:00 0\n"]
    ops._one_runtime(one)
    with pytest.raises(RuntimeError, match="before the first Model"):
        ops._one_runtime(one + [line("/site/torch/lib/libamdhip64.so")])
