"""Operators on a pool over the caller's memory: cache writes and attention give the bits that they give on a pool of the library's own,
before and after sequences branch and the pool is compacted, whatever type the process's own pools have."""
import ctypes as C

import numpy as np
import pytest

from nvllm_amd import capi
from tests import util
from tests.test_gpu_sequence_memory import pointers

pytestmark = pytest.mark.gpu
L, BS, NB, S = 3, 16, 60, 512


class Attached(util.Pool):
    def __init__(self, hip, elem, kv_heads, head_dim):
        self.lib, self.mgr, self.geom, self.tables = hip, capi.KVCacheManager(), (L, kv_heads, head_dim), []
        self.size = L * NB * BS * kv_heads * head_dim * elem
        self.own = [hip.empty_device(self.size) for _ in range(2)]
        assert hip.nvllm_attach_kv_pool(C.byref(self.mgr), BS, NB, L, kv_heads, head_dim, elem, *self.own) == 0

    def memory(self):
        return [self.lib.to_host(p, (self.size,), np.uint8) for p in (self.mgr.pool_k, self.mgr.pool_v)]

    def close(self):
        before = self.memory()
        self.lib.free_kv_cache_manager(C.byref(self.mgr))
        for p, x in zip(self.own, before):
            np.testing.assert_array_equal(self.lib.to_host(p, (self.size,), np.uint8), x)   # still the caller's
            self.lib.free(p)


class Library(Attached):
    def __init__(self, hip, elem, kv_heads, head_dim):
        self.lib, self.mgr, self.geom, self.tables = hip, capi.KVCacheManager(), (L, kv_heads, head_dim), []
        self.size = L * NB * BS * kv_heads * head_dim * elem
        hip.nvllm_set_kv_elem_bytes(elem)
        hip.init_kv_cache_manager(C.byref(self.mgr), BS, NB, L, kv_heads, head_dim)
        hip.nvllm_set_kv_elem_bytes(4)

    def close(self):
        self.lib.free_kv_cache_manager(C.byref(self.mgr))


def story(hip, pool, H, KVH, hd):
    """Two prompts, a step, a fork in the middle of a block, tokens of each branch, a sequence's end, compaction, a step; what attention gave."""
    r = np.random.Generator(np.random.PCG64(hd))
    out = []
    m = C.byref(pool.mgr)

    def run(parts):
        pos = [p for _, a, b in parts for p in range(a, b)]
        sid = [s for s, a, b in parts for _ in range(a, b)]
        for s, _, b in parts:
            pool.grow(s, b)
        for layer in range(L):
            k, v = (r.standard_normal((len(pos), KVH * hd)).astype(np.float32) for _ in range(2))
            q = r.standard_normal((len(pos), H * hd)).astype(np.float32)
            util.op_kv_write_batch(hip, pool, k, v, layer, pos, sid, KVH, hd)
            out.append(util.op_paged_attention_batch(hip, pool, q, layer, pos, sid, S, H, KVH, hd))

    for _ in range(4):
        pool.new_table(S // BS)
    table = [t for t, _ in pool.tables]
    run([(0, 0, 100), (1, 0, 70)])
    run([(0, 100, 101), (1, 70, 71)])
    assert hip.nvllm_fork_tables(m, C.byref(table[1]), 71, pointers([table[2], table[3]]), 2) == 0
    run([(1, 71, 72), (2, 71, 90), (3, 71, 72)])
    assert hip.nvllm_free_table(m, C.byref(table[0])) == 0
    assert hip.nvllm_compact_blocks(m, pointers(table[1:]), 3) > 0
    run([(2, 90, 91), (1, 72, 75), (3, 72, 73)])
    return out


@pytest.mark.parametrize("elem", [4, 2], ids=["fp32", "fp16"])
@pytest.mark.parametrize("hd,H,KVH", [(64, 8, 2), (48, 6, 6), (128, 4, 4)])
def test_like_a_pool_of_the_librarys(hip, elem, hd, H, KVH):
    a, b = Attached(hip, elem, KVH, hd), Library(hip, elem, KVH, hd)
    want = story(hip, b, H, KVH, hd)
    hip.nvllm_set_kv_elem_bytes(6 - elem)   # (what new pools of the process would have)
    try:
        got = story(hip, a, H, KVH, hd)
    finally:
        hip.nvllm_set_kv_elem_bytes(4)
    assert len(got) == len(want) == 4 * L
    for x, y in zip(got, want):
        np.testing.assert_array_equal(x, y)
        assert np.isfinite(x).all() and np.abs(x).max() > 0
    for x, y in zip(a.memory(), b.memory()):
        np.testing.assert_array_equal(x, y)
    assert [t.block_indices[:t.num_blocks] for t, _ in a.tables] == [t.block_indices[:t.num_blocks] for t, _ in b.tables]
    a.close()
    b.close()
