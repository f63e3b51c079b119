"""The caller's memory is the caller's again when its pool has been released: what was enqueued on it is over."""
import ctypes as C

import pytest

from nvllm_amd import capi
from tests import hip_standin


def test_a_release_waits(tmp_path):
    hip_standin.run(tmp_path, """
def attached():
    m = capi.KVCacheManager()
    assert lib.nvllm_attach_kv_pool(C.byref(m), 16, 8, 2, 2, 32, 4, 0x100000, 0x100000000) == 0
    return m
m = attached()
assert lib.nvllm_copy_blocks(C.byref(m), ints([0, 1]), ints([2, 3]), 2) == 0 and gpu.standin_launches() == 1
before = gpu.standin_waits()
lib.free_kv_cache_manager(C.byref(m))
assert gpu.standin_waits() > before and gpu.standin_taken() == 0
m = attached()
before = gpu.standin_waits()
gpu.standin_capture(1)      # a captured stream cannot be waited for: nothing runs on it yet
lib.free_kv_cache_manager(C.byref(m))
assert gpu.standin_waits() == before
""")


@pytest.mark.gpu
def test_a_release_waits_for_copies(hip):
    rtl = C.CDLL("libamdhip64.so")
    blocks, layers, size = 64, 16, 1 << 29          # half a GB each of keys and values
    own = [C.c_void_p(), C.c_void_p()]
    m = capi.KVCacheManager()
    assert all(hip.device_malloc(C.byref(p), size) == 0 for p in own)
    assert hip.nvllm_attach_kv_pool(C.byref(m), 16, blocks, layers, 8, size // (blocks * layers * 16 * 8 * 4), 4, *own) == 0
    frm, to = capi.ints(range(32)), capi.ints(range(32, 64))
    for _ in range(100):                            # 100 times 1 GB read and written: over 15 ms
        assert hip.nvllm_copy_blocks(C.byref(m), frm, to, 32) == 0
    hip.free_kv_cache_manager(C.byref(m))
    assert rtl.hipStreamQuery(C.c_void_p(hip.nvllm_stream())) == 0
    for p in own:
        hip.free(p)
