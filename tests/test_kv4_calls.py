"""Calls of the 4-bit operators that are not refused, and what they need, on the CPU."""
import pytest

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
