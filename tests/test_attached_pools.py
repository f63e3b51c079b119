"""Pools over the caller's memory: who may let go of what, without a GPU.  Child processes: a release that reached for memory which is not
the library's would end them."""
import os
import subprocess
import sys

import pytest

from nvllm_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEAD = """
import ctypes as C
from nvllm_amd import capi
lib = capi.load_hip()
def attach(at=0x100000, blocks=8, into=None):
    m = into or capi.KVCacheManager()
    assert lib.nvllm_attach_kv_pool(C.byref(m), 16, blocks, 2, 2, 32, 4, at, at + 0x800000) == 0
    return m
def table(m, n=0):
    room = (C.c_int * 8)(*[lib.alloc_block(C.byref(m)) for _ in range(n)])
    t = capi.BlockTable(C.cast(room, capi.c_int_p), n)
    t.keep = room
    return t
def fork(m, t, positions):
    to = table(m)
    return lib.nvllm_fork_tables(C.byref(m), C.byref(t), positions, (C.POINTER(capi.BlockTable) * 1)(C.pointer(to)), 1), to
def users(m, n):
    return [lib.nvllm_block_users(C.byref(m), i) for i in range(n)]
def release(m):
    lib.free_kv_cache_manager(C.byref(m))
    assert not m.pool_k and not m.pool_v and not m.free_block_indices
"""


def run(body):
    r = subprocess.run([sys.executable, "-c", HEAD + body], capture_output=True, text=True, timeout=100, env=dict(os.environ, PYTHONPATH=ROOT + os.pathsep + os.environ.get("PYTHONPATH", "")))
    assert r.returncode == 0, r.stderr[-1000:]


@pytest.mark.parametrize("order", [(0, 1), (1, 0)], ids=["the earlier first", "the later first"])
def test_memory_that_is_attached_twice_stays_the_callers(order):
    run("""
m = [attach(), attach()]
for i in %r:
    release(m[i])
m = attach()
assert fork(m, table(m, 2), 32)[0] == 0 and users(m, 3) == [2, 2, 0]
release(m)
""" % (order,))


def test_a_manager_that_attaches_again():
    run("""
m = attach()
attach(0x9100000, 4, m)
assert m.num_blocks == 4 and fork(m, table(m, 1), 16)[0] == 0
release(m)
release(attach(blocks=3))
""")


def test_counts_are_the_managers_own():
    """Memory that is attached again is the later manager's; what the earlier one has counted stays right until it is released."""
    run("""
a = attach()
t = table(a, 3)
rc, child = fork(a, t, 48)
assert rc == 0 and users(a, 4) == [2, 2, 2, 0]
b = attach()
assert users(a, 4) == [2, 2, 2, 0] and users(b, 4) == [0] * 4
assert fork(a, t, 48)[0] == -2 and lib.nvllm_compact_blocks(C.byref(a), None, 0) == -2 and lib.nvllm_copy_blocks(C.byref(a), capi.ints([0]), capi.ints([0]), 1) == -2
assert lib.nvllm_free_table(C.byref(a), C.byref(t)) == 0 and users(a, 4) == [1, 1, 1, 0] and a.free_blocks_count == 5
u = table(b, 2)
assert fork(b, u, 32)[0] == 0 and users(b, 3) == [2, 2, 0] and users(a, 4) == [1, 1, 1, 0]
release(a)
assert users(b, 3) == [2, 2, 0] and fork(b, u, 16)[0] == 0 and users(b, 3) == [3, 2, 0]
release(b)
""")


def test_a_free_stack_without_memory():
    """The host's own memory: a pool whose free stack the system does not give."""
    run("""
import resource
resource.setrlimit(resource.RLIMIT_AS, (8 << 30, 8 << 30))
m = capi.KVCacheManager()
assert lib.nvllm_attach_kv_pool(C.byref(m), 1, 0x7fffffff, 1, 1, 1, 4, 0x100000, 0x100000000) == -5
assert not m.free_block_indices and not m.pool_k
release(attach(blocks=1000))
""")
