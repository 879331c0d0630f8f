"""Calls of the 4-bit operators that are not refused, and what they need, on the CPU."""
import os
import re

import pytest

from conftest import ROOT
from test_kv4_plan import be, call  # noqa: F401  (be: a fixture)


def attend(be, **more):
    """what an attention call asks for and answers where it has nothing to do: (workspace, status)"""
    from tinygpt_amd.ffi import Kv4BatchArg, Kv4CacheArg, Kv4RowsArg
    a = dict(pages=4, table=4096, table_stride=3, table_len=3, seqs=2, kv_heads=2, head_dim=64, pool=4096, entries=2, max_count=1, tokens=2, offsets=None, start=4096, heads=4, window=0, keys=300)
    a.update(more)
    c = Kv4CacheArg(a["pool"], a["pages"], a["table"], a["table_stride"], a["table_len"], a["seqs"], a["kv_heads"], a["head_dim"])
    return be.kv4_attend_workspace(c, Kv4BatchArg(a["entries"], a["max_count"], a["tokens"], None, a["start"], a["offsets"]), a["heads"], a["window"], a["keys"], 0)


@pytest.mark.parametrize("heads", [2, 8, 32])
def test_batches_of_many_tokens_have_a_plan(be, heads):  # noqa: F811
    """64 prompts of 1024 tokens, max_count left at all of them: every entry is short"""
    assert attend(be, entries=64, seqs=64, tokens=65536, max_count=65536, offsets=4096, heads=heads, keys=1024) >= 0
    assert attend(be, entries=1, seqs=1, tokens=130000, max_count=130000, offsets=4096, heads=heads, keys=131072) >= 0


@pytest.mark.parametrize("name", ["append", "read", "attend"])
def test_batches_without_tokens_need_no_buffers(be, name):  # noqa: F811
    """entries that bring nothing (a tensor of no numbers has no address)"""
    assert call(be, name, entries=3, tokens=0, max_count=0, offsets=4096, data=None) == 0
    assert call(be, name, entries=3, tokens=0, max_count=16, offsets=4096, data=None) == 0
    assert call(be, name, entries=3, tokens=7, max_count=0, offsets=4096) == 0
    assert call(be, name, entries=3, tokens=-1, max_count=0, offsets=4096, data=None) == 1
    assert call(be, name, entries=3, tokens=0, max_count=0, offsets=4096, data=None, start=None) == 1


def test_copies_of_pools_without_pages(be):  # noqa: F811
    for src, dst in [(0, 4), (4, 0), (0, 0)]:
        assert be.copy_pages(4096 if src else None, src, 4096, 8192 if dst else None, dst, 4096, 2, 256, 4096, 4096, 2, 0, None) == 0


@pytest.mark.parametrize("window", [0, 100, 5000])
@pytest.mark.parametrize("max_count,entries,heads", [(1, 1, 8), (1, 32, 8), (5, 3, 4), (300, 1, 8)])
def test_the_keys_of_a_page_need_one_workspace(be, max_count, entries, heads, window):  # noqa: F811
    """ops.kv4_attend looks a workspace up by whole pages of max_keys: what the library says for max_keys itself"""
    from tinygpt_amd.ops import _whole_pages
    needs = set()
    for keys in [0, 1, 2, 127, 128, 129, 255, 256, 257, 700, 1023, 1024, 1025, 4095, 4097, 30000, 131071, 131072, 2 ** 31 - 129, 2 ** 31 - 128, 2 ** 31 - 127, 2 ** 31 - 1]:
        size = dict(entries=entries, seqs=entries, tokens=entries * max_count, max_count=max_count, offsets=4096, heads=heads, window=window)
        needs.add(attend(be, keys=keys, **size))
        assert attend(be, keys=keys, **size) == attend(be, keys=_whole_pages(keys), **size) >= 0, keys
    assert len(needs) > 1 or window or max_count == 300


def test_a_generation_looks_its_workspace_up_once_a_page():
    from tinygpt_amd.ops import _whole_pages
    assert len({_whole_pages(k) for k in range(1, 1025)}) == 8
    assert _whole_pages(0) == 0 and _whole_pages(-1) == 0 and _whole_pages(2 ** 40) == 2 ** 31 - 1


def test_bytes_in_lds_are_aligned_for_wider_reads():
    """arrays of bytes that a kernel of kv4.h holds in LDS are read as words: each says its alignment"""
    with open(os.path.join(ROOT, "tinygpt_amd", "csrc", "kernels", "kv4.h")) as f:
        arrays = re.findall(r"^.*__shared__.*unsigned char .*$", f.read(), re.M)
    assert len(arrays) == 2 and all("aligned(16)" in a for a in arrays), arrays


def test_outputs_that_lie_on_each_other_are_refused(be):  # noqa: F811
    """a stride of 0 in an output of several tokens or heads; inputs may repeat"""
    from tinygpt_amd.ffi import Kv4BatchArg, Kv4CacheArg, Kv4RowsArg
    c, b = Kv4CacheArg(4096, 4, 4096, 3, 3, 2, 2, 64), Kv4BatchArg(2, 1, 2, None, 4096, None)
    good = Kv4RowsArg(4096, 1, 256, 64)
    for token, head in [(0, 64), (256, 0), (0, 0)]:
        bad = Kv4RowsArg(4096, 1, token, head)
        assert be.kv4_read(c, b, bad, good, 0, None) == 1 and be.kv4_read(c, b, good, bad, 0, None) == 1
        assert be.kv4_attend(c, b, good, 4, good, good, 0.125, 0, 300, bad, 4096, 1 << 40, 0, None) == 1
        assert b"share memory" in be.op_last_error()


def test_copies_into_layers_that_share_memory_are_refused(be):  # noqa: F811
    """pages of one layer of the destination would be another's; a source may repeat (one layer into several)"""
    for stride, pages, layers, status in [(0, 4, 2, 1), (256 * 3, 4, 2, 1), (256 * 4 - 16, 4, 2, 1), (256, 2, 9, 1)]:
        assert be.copy_pages(4096, 4, 1024, 8192, pages, stride, layers, 256, 4096, 4096, 2, 0, None) == status, stride
        assert b"share memory" in be.op_last_error()
