"""A pool of the library's at an address that was attached once and never released: nothing of the old pool reaches the new one.  A stand-in
takes the runtime's place, whose addresses are known beforehand."""
import pytest

from tests import hip_standin


@pytest.mark.parametrize("kind", ["kv", "latent", "window"])
def test_a_pool_where_another_was_attached(tmp_path, kind):
    hip_standin.run(tmp_path, """
make = dict(kv=lambda m: lib.init_kv_cache_manager(m, 16, 8, 2, 2, 32), latent=lambda m: lib.nvllm_latent_pool_init(m, 16, 8, 20, 12, 4),
            window=lambda m: lib.nvllm_window_pool_init(m, 16, 8, 2, 32, 32, 4))[%r]
def table(m, n):
    at = (C.c_int * 8)(*[lib.alloc_block(C.byref(m)) for _ in range(n)])
    t = capi.BlockTable(C.cast(at, capi.c_int_p), n)
    t.keep = at
    return t
def fork(m, t, positions):
    to = table(m, 0)
    return lib.nvllm_fork_tables(C.byref(m), C.byref(t), positions, (C.POINTER(capi.BlockTable) * 1)(C.pointer(to)), 1)
def users(m):
    return [lib.nvllm_block_users(C.byref(m), i) for i in range(4)]
p = C.c_void_p()
assert lib.device_malloc(C.byref(p), 100) == 0
step = 1 << 24                                   # from one of the stand-in's addresses to the next
lib.device_free(p)
free = gpu.standin_taken()
old = capi.KVCacheManager()
assert lib.nvllm_attach_kv_pool(C.byref(old), 16, 8, 2, 2, 32, 4, p.value + step, p.value + 9 * step) == 0
assert fork(old, table(old, 3), 48) == 0 and users(old) == [2, 2, 2, 0]
new = capi.KVCacheManager()
make(C.byref(new))
assert new.pool_k == p.value + step
t = table(new, 3)
assert users(new) == [1, 1, 1, 0] and users(old) == [2, 2, 2, 0]
assert lib.nvllm_free_table(C.byref(new), C.byref(t)) == 0 and new.free_blocks_count == 8
t = table(new, 2)
assert fork(new, t, 20) == 0 and users(new) == [2, 1, 1, 0]
taken = gpu.standin_taken()
lib.free_kv_cache_manager(C.byref(old))          # the caller's memory, whatever lies there now
assert gpu.standin_taken() == taken and users(new) == [2, 1, 1, 0] and fork(new, t, 16) == 0
lib.free_kv_cache_manager(C.byref(new))
assert gpu.standin_taken() == free
""" % kind)
