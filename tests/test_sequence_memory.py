"""Tables of branching sequences: the host's bookkeeping and its refusals, without a GPU (no copy is reached here)."""
import ctypes as C

import numpy as np
import pytest

from nvllm_amd import capi

BAD_ARGUMENT, BAD_SIZE, BAD_INDEX, NO_BLOCKS = -1, -2, -3, -4


@pytest.fixture(scope="module")
def lib():
    return capi.load_hip()


class Pool:
    """A pool over addresses that nothing reads."""
    next = 0x100000

    def __init__(self, lib, blocks=12, **kw):
        self.lib, self.m = lib, capi.KVCacheManager()
        a = dict(dict(block_size=16, num_blocks=blocks, n_layers=2, n_kv_heads=2, head_dim=32, elem_bytes=4), **kw)
        Pool.next += 0x1000000
        rc = lib.nvllm_attach_kv_pool(C.byref(self.m), *a.values(), Pool.next, Pool.next + 0x800000)
        assert rc == 0
        self.keep = []

    def table(self, blocks=(), room=16):
        at = (C.c_int * room)(*blocks)
        t = capi.BlockTable(C.cast(at, capi.c_int_p), len(blocks))
        self.keep += [at, t]
        return t

    def take(self, n):
        return self.table([self.lib.alloc_block(C.byref(self.m)) for _ in range(n)])

    def fork(self, t, positions, n):
        to = [self.table() for _ in range(n)]
        return self.lib.nvllm_fork_tables(C.byref(self.m), C.byref(t), positions, pointers(to), n), to

    def users(self, b):
        return self.lib.nvllm_block_users(C.byref(self.m), b)

    def free(self, t):
        return self.lib.nvllm_free_table(C.byref(self.m), C.byref(t))

    def compact(self, tables):
        return self.lib.nvllm_compact_blocks(C.byref(self.m), pointers(tables), len(tables))

    def stack(self):
        return self.m.free_block_indices[:self.m.free_blocks_count]


def pointers(tables):
    return (C.POINTER(capi.BlockTable) * max(1, len(tables)))(*[C.pointer(t) for t in tables])


def blocks(t):
    return t.block_indices[:t.num_blocks]


def test_a_pool_of_the_callers_memory_starts_like_any_other(lib):
    p = Pool(lib)
    assert p.stack() == list(range(11, -1, -1)) and (p.m.block_size, p.m.num_blocks) == (16, 12)
    lib.free_kv_cache_manager(C.byref(p.m))   # leaves the memory alone
    assert not p.m.pool_k and not p.m.free_block_indices


def test_whole_blocks_are_shared_until_their_last_user_frees_them(lib):
    p = Pool(lib)
    t = p.take(3)
    rc, (a, b) = p.fork(t, 48, 2)
    assert rc == 0 and blocks(a) == blocks(b) == blocks(t) == [0, 1, 2]
    assert [p.users(i) for i in range(4)] == [3, 3, 3, 0]
    rc, (c,) = p.fork(a, 32, 1)
    assert rc == 0 and blocks(c) == [0, 1] and [p.users(i) for i in range(3)] == [4, 4, 3]
    before = p.stack()
    assert p.free(t) == 0 and t.num_blocks == 0 and p.stack() == before
    assert p.free(b) == 0 and p.free(c) == 0 and p.stack() == before
    assert [p.users(i) for i in range(3)] == [1, 1, 1]
    assert p.free(a) == 0 and p.stack() == before + [2, 1, 0]
    lib.free_block(C.byref(p.m), 5)   # (as before: a full stack takes nothing)
    assert p.m.free_blocks_count == 12 and [p.users(i) for i in range(12)] == [0] * 12


def test_forks_of_nothing(lib):
    p = Pool(lib)
    t = p.take(1)
    rc, (a,) = p.fork(t, 0, 1)
    assert rc == 0 and a.num_blocks == 0 and p.users(0) == 1
    assert p.fork(t, 16, 0)[0] == 0
    assert p.fork(p.table(), 0, 2)[0] == 0


def test_forks_that_are_refused_change_nothing(lib):
    p = Pool(lib, 4)
    t = p.take(3)
    stack = p.stack()

    def refused(rc, what):
        assert rc == what and p.stack() == stack and [p.users(i) for i in range(4)] == [1, 1, 1, 0]
    refused(p.fork(t, 49, 1)[0], BAD_INDEX)                  # more positions than blocks
    refused(p.fork(t, 40, 2)[0], NO_BLOCKS)                  # two copies of the last, one block free
    refused(p.fork(t, -1, 1)[0], BAD_ARGUMENT)
    refused(p.fork(t, 16, -1)[0], BAD_ARGUMENT)
    refused(p.fork(p.table([0, 3]), 32, 1)[0], BAD_INDEX)    # a free block
    refused(p.fork(p.table([0, 0]), 32, 1)[0], BAD_INDEX)
    refused(p.fork(p.table([0, 4]), 32, 1)[0], BAD_INDEX)
    refused(p.fork(p.table([-1]), 16, 1)[0], BAD_INDEX)
    to = p.table()
    f = lib.nvllm_fork_tables
    m = C.byref(p.m)
    refused(f(m, C.byref(t), 16, pointers([to, to]), 2), BAD_ARGUMENT)
    refused(f(m, C.byref(t), 16, pointers([t]), 1), BAD_ARGUMENT)
    refused(f(m, C.byref(t), 16, None, 1), BAD_ARGUMENT)
    refused(f(m, None, 16, pointers([to]), 1), BAD_ARGUMENT)
    refused(f(None, C.byref(t), 16, pointers([to]), 1), BAD_ARGUMENT)
    refused(f(m, C.byref(t), 16, pointers([capi.BlockTable(None, 0)]), 1), BAD_ARGUMENT)
    assert to.num_blocks == 0


def test_a_pool_that_the_library_does_not_know(lib):
    m = capi.KVCacheManager()
    stack = (C.c_int * 4)(3, 2, 1, 0)
    m.block_size, m.num_blocks, m.free_blocks_count, m.free_block_indices, m.pool_k = 16, 4, 2, C.cast(stack, capi.c_int_p), 0x77000000
    at = (C.c_int * 1)(0)
    t = capi.BlockTable(C.cast(at, capi.c_int_p), 1)
    one = capi.ints([0])
    assert lib.nvllm_copy_blocks(C.byref(m), one, capi.ints([1]), 1) == BAD_SIZE
    assert lib.nvllm_compact_blocks(C.byref(m), pointers([t]), 1) == BAD_SIZE
    assert lib.nvllm_fork_tables(C.byref(m), C.byref(t), 16, pointers([capi.BlockTable(C.cast(at, capi.c_int_p), 0)]), 1) == BAD_SIZE


def test_compaction_without_moves(lib):
    """Blocks in use already lie in front; the free stack is in order again."""
    p = Pool(lib, 8)
    a, b = p.take(2), p.take(2)
    lib.free_block(C.byref(p.m), 2)
    lib.free_block(C.byref(p.m), 3)
    b.num_blocks = 0
    assert p.stack() == [7, 6, 5, 4, 2, 3]
    assert p.compact([a, b]) == 0 and p.stack() == [7, 6, 5, 4, 3, 2] and blocks(a) == [0, 1]
    assert p.compact([]) == 0


def test_compaction_leaves_what_it_cannot_rewrite(lib):
    """A block that no given table has, and one whose other users are not given, stay where they are."""
    p = Pool(lib, 8)
    a, b = p.take(3), p.take(3)          # 0 1 2, 3 4 5
    rc, (c,) = p.fork(b, 48, 1)
    assert rc == 0 and p.free(a) == 0    # 3 4 5 in use, by two tables
    assert p.compact([b]) == 0 and p.compact([c]) == 0 and p.compact([]) == 0
    assert blocks(b) == blocks(c) == [3, 4, 5] and p.stack() == [7, 6, 2, 1, 0]


def test_compactions_that_are_refused_change_nothing(lib):
    p = Pool(lib, 8)
    a, b = p.take(2), p.take(2)
    assert p.free(a) == 0
    stack = p.stack()

    def refused(rc, what):
        assert rc == what and p.stack() == stack and blocks(b) == [2, 3]
    refused(p.compact([b, p.table([0])]), BAD_INDEX)         # a free block
    refused(p.compact([p.table([8])]), BAD_INDEX)
    refused(p.compact([p.table([-1])]), BAD_INDEX)
    refused(p.compact([b, b]), BAD_ARGUMENT)
    refused(lib.nvllm_compact_blocks(C.byref(p.m), None, 1), BAD_ARGUMENT)
    refused(lib.nvllm_compact_blocks(C.byref(p.m), (C.POINTER(capi.BlockTable) * 1)(), 1), BAD_ARGUMENT)
    refused(lib.nvllm_compact_blocks(None, pointers([b]), 1), BAD_ARGUMENT)
    p.m.free_block_indices[0] = p.m.free_block_indices[1]   # a stack that holds a block twice
    assert p.compact([b]) == BAD_INDEX


def test_tables_that_cannot_be_freed(lib):
    p = Pool(lib, 4)
    assert p.free(p.table([0, 4])) == BAD_INDEX and lib.nvllm_free_table(C.byref(p.m), None) == BAD_ARGUMENT
    assert lib.nvllm_free_table(None, C.byref(p.table())) == BAD_ARGUMENT
    assert p.users(4) == BAD_ARGUMENT and p.users(-1) == BAD_ARGUMENT
    assert p.m.free_blocks_count == 4


def test_copies_that_are_refused(lib):
    p = Pool(lib, 8)
    m = C.byref(p.m)

    def copy(f, t):
        return lib.nvllm_copy_blocks(m, capi.ints(f), capi.ints(t), len(f)), lib.nvllm_copy_states(0x1000, 64, 2, 8, capi.ints(f), capi.ints(t), len(f))
    for f, t in (([0], [8]), ([8], [0]), ([-1], [0]), ([0], [-1]), ([0, 1], [2, 2]), ([0, 0], [0, 0])):
        assert copy(f, t) == (BAD_INDEX, BAD_INDEX)
    one = capi.ints([0])
    assert lib.nvllm_copy_blocks(m, None, one, 1) == lib.nvllm_copy_blocks(m, one, None, 1) == lib.nvllm_copy_blocks(None, one, one, 1) == BAD_ARGUMENT
    assert lib.nvllm_copy_blocks(m, one, one, -1) == BAD_ARGUMENT
    s = lib.nvllm_copy_states
    assert s(None, 64, 1, 8, one, one, 1) == s(0x1000, 64, -1, 8, one, one, 1) == s(0x1000, 64, 1, -1, one, one, 1) == s(0x1000, 64, 1, 8, one, one, -1) == BAD_ARGUMENT
    assert s(0x1000, 1 << 45, 1, 8, one, one, 1) == BAD_SIZE
    # nothing to do: no slot, no array, a slot onto itself
    assert s(None, 64, 1, 8, None, None, 0) == s(0x1000, 0, 1, 8, one, one, 1) == s(0x1000, 64, 0, 8, one, one, 1) == 0
    assert copy([3, 5], [3, 5]) == (0, 0)


@pytest.mark.parametrize("over,what", [
    (dict(block_size=0), BAD_ARGUMENT), (dict(num_blocks=0), BAD_ARGUMENT), (dict(n_layers=0), BAD_ARGUMENT), (dict(n_kv_heads=-1), BAD_ARGUMENT), (dict(head_dim=0), BAD_ARGUMENT),
    (dict(k=None), BAD_ARGUMENT), (dict(v=None), BAD_ARGUMENT), (dict(k=0x1008), BAD_ARGUMENT), (dict(v=0x1000), BAD_ARGUMENT),
    (dict(elem_bytes=1), BAD_SIZE), (dict(elem_bytes=2, block_size=32), BAD_SIZE), (dict(elem_bytes=2, head_dim=24), BAD_SIZE), (dict(num_blocks=1 << 28), BAD_SIZE)], ids=str)
def test_pools_that_cannot_be_attached(lib, over, what):
    a = dict(dict(block_size=16, num_blocks=4, n_layers=1, n_kv_heads=1, head_dim=32, elem_bytes=4, k=0x1000, v=0x2000), **over)
    assert lib.nvllm_attach_kv_pool(C.byref(capi.KVCacheManager()), *a.values()) == what
    assert lib.nvllm_attach_kv_pool(None, *dict(a, block_size=16).values()) == BAD_ARGUMENT
