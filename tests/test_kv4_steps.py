"""The workspace of a model's steps over a 4-bit cache (tinygpt_amd/csrc/kv4_plan.h, kv4_step_floats) holds the records of every step, compiled with the host compiler."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT

SOURCE = r"""
#include "kv4_plan.h"
using namespace tgx;
// the keys at which some step's records do not fit, 0: none; *divided: steps that divide the keys
extern "C" long long misfit(int max_batch, int heads, int kv_heads, int hd, long long max_ctx, int cus, long long* divided) {
  const size_t have = kv4_step_floats(max_batch, heads, kv_heads, hd, max_ctx, cus);
  *divided = 0;
  for (int R = 1; R <= (max_batch < 4 ? 4 : max_batch); R++)
    for (long long keys = 1; keys <= max_ctx; keys += keys < 300 ? 1 : keys / 37) {
      const Kv4Plan p = kv4_plan(R, 1, kv_heads, heads / kv_heads, hd, 0, kv4_bucket(keys), cus);
      *divided += p.splits > 1;
      if (kv4_part_floats(p, (long long)R * heads, hd) > have) return keys;
    }
  return 0;
}
extern "C" int bucket(long long keys) { return kv4_bucket(keys); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv4steps")
    src, so = d / "steps.cpp", d / "libsteps.so"
    src.write_text(SOURCE)
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "tinygpt_amd", "csrc"), str(src), "-o", str(so)])
    lib = ctypes.CDLL(str(so))
    lib.misfit.argtypes = [ctypes.c_int] * 4 + [ctypes.c_longlong, ctypes.c_int, ctypes.POINTER(ctypes.c_longlong)]
    lib.misfit.restype = ctypes.c_longlong
    lib.bucket.argtypes = [ctypes.c_longlong]
    return lib


@pytest.mark.parametrize("cus", [64, 256, 304])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 64), (32, 8, 64), (32, 8, 128), (14, 2, 64), (12, 12, 64), (16, 1, 128), (64, 8, 128)])
def test_every_step_fits(lib, heads, kv_heads, hd, cus):
    divided = ctypes.c_longlong()
    for max_batch in (1, 3, 8, 40, 128):
        for max_ctx in (1, 255, 768, 1024, 1500, 4096, 131072):
            assert lib.misfit(max_batch, heads, kv_heads, hd, max_ctx, cus, ctypes.byref(divided)) == 0, (max_batch, max_ctx)
            assert max_ctx < 4096 or divided.value > 0


def test_buckets(lib):
    for keys, want in [(0, 256), (1, 256), (256, 256), (257, 512), (2048, 2048), (2049, 4096), (2 ** 40, 2 ** 30)]:
        assert lib.bucket(keys) == want
