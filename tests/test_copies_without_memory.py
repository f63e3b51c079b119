"""Calls whose workspace finds no memory are refused before anything is enqueued or changed; a stand-in takes the runtime's place."""
from tests import hip_standin

NO_MEMORY = -5
CALLS = """
def refused(call):
    gpu.standin_forget()
    assert call() == -5
    assert gpu.standin_launches() == 0, launches()
def passes(call):
    gpu.standin_forget()
    assert call() == 0 and gpu.standin_launches() > 0
"""


def test_copies(tmp_path):
    hip_standin.run(tmp_path, CALLS + """
n = 4000
frm, to = ints(np.arange(n)), ints(np.arange(n) + n)
states = lambda: lib.nvllm_copy_states(0x1000, 64, 2, 2 * n, frm, to, n)
m = capi.KVCacheManager()
assert lib.nvllm_attach_kv_pool(C.byref(m), 16, 2 * n, 2, 2, 32, 4, 0x100000, 0x100000000) == 0
gpu.standin_memory(1000)
refused(states)
refused(lambda: lib.nvllm_copy_blocks(C.byref(m), frm, to, n))
gpu.standin_memory(1 << 30)
passes(states)
passes(lambda: lib.nvllm_copy_blocks(C.byref(m), frm, to, n))
""")


def test_forks_and_compaction_change_nothing(tmp_path):
    hip_standin.run(tmp_path, CALLS + """
n = 1200
m = capi.KVCacheManager()
assert lib.nvllm_attach_kv_pool(C.byref(m), 16, 2 * n, 2, 2, 32, 4, 0x100000, 0x100000000) == 0
def table(k, room=4):
    at = (C.c_int * room)(*[lib.alloc_block(C.byref(m)) for _ in range(k)])
    t = capi.BlockTable(C.cast(at, capi.c_int_p), k)
    t.keep = at
    return t
def pointers(ts):
    return (C.POINTER(capi.BlockTable) * len(ts))(*[C.pointer(t) for t in ts])
def stack():
    return m.free_block_indices[:m.free_blocks_count]
gone = table(600, 600)
parent = table(2)
children = [table(0) for _ in range(n)]
before = stack()
gpu.standin_memory(1000)
refused(lambda: lib.nvllm_fork_tables(C.byref(m), C.byref(parent), 20, pointers(children), n))
assert stack() == before and lib.nvllm_block_users(C.byref(m), 600) == 1 and all(t.num_blocks == 0 for t in children)
gpu.standin_memory(1 << 30)
passes(lambda: lib.nvllm_fork_tables(C.byref(m), C.byref(parent), 20, pointers(children), n))
assert lib.nvllm_block_users(C.byref(m), 600) == n + 1 and [c.block_indices[1] for c in children] == before[::-1][:n]
assert lib.nvllm_free_table(C.byref(m), C.byref(gone)) == 0
lib.free_ops()                   # (the workspaces are given back)
gpu.standin_memory(1000)
before = stack()
tables = pointers([parent] + children)
refused(lambda: lib.nvllm_compact_blocks(C.byref(m), tables, n + 1))
assert stack() == before and [c.block_indices[1] for c in children] == list(range(602, 602 + n)) and lib.nvllm_block_users(C.byref(m), 600) == n + 1
gpu.standin_memory(1 << 30)
gpu.standin_forget()
assert lib.nvllm_compact_blocks(C.byref(m), tables, n + 1) == 600 and gpu.standin_launches() > 0
""")
