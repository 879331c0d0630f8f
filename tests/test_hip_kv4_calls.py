"""Calls of the 4-bit cache, its operators and the forks that one might not think of: what a refusal leaves, sizes of zero, large batches, pending tokens."""
import ctypes

import numpy as np
import pytest
import torch   # here, not in a test: before any module's test loads the library, which then shares torch's HIP runtime

from test_hip_kv4_model import ids, make
from tinygpt_amd.ffi import GREEDY, TgxError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from tinygpt_amd.ffi import product_backend
    return product_backend()


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


# ---- models ----------------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("missing", ["keys", "values"])
def test_a_refused_write_leaves_a_fork_its_shared_blocks(missing, hip):
    m, _ = make("llama_tiny", hip, "bf16", 4, max_batch=2, budget=1024)
    m.forward_row(0, ids(np.random.default_rng(1), 300, m.desc.vocab)[0])
    m.fork_row(0, 1)
    free = m.get_option("kv.free_tokens")
    k, _ = m.read_kv(0, 0)
    p = k.ctypes.data_as(ctypes.POINTER(ctypes.c_float))
    with pytest.raises(TgxError):
        m._check(m.be.write_kv(m._ctx, 0, 0, None if missing == "keys" else p, None if missing == "values" else p, 300))
    assert m.get_option("kv.free_tokens") == free
