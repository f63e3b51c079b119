"""A copy of more workgroups than one grid takes: the rest goes in launches of its own."""
import ctypes as C

import numpy as np
import pytest

from nvllm_amd import capi

pytestmark = pytest.mark.gpu


def test_odd_slots_behind_the_first_grid(hip):
    """Slots of 2^30 + 1 bytes, a byte a thread: 2,097,153 pieces of nine programs, more than a grid takes."""
    slot, n = (1 << 30) + 1, 9
    pieces = -(-slot // 512)
    assert pieces * n * 256 >= 1 << 32
    edge = 0xffffffff // 256 // n * 512   # the first byte of a slot that the second launch moves
    p = C.c_void_p()
    assert hip.device_malloc(C.byref(p), 2 * n * slot) == 0
    r = np.random.Generator(np.random.PCG64(3))
    windows = [(0, 3000), (edge - 1500, edge + 1500), (slot - 3000, slot)]
    frm, to = np.arange(n), n + (np.arange(n) * 2) % n
    want = {}
    for i, f in enumerate(frm):
        for a, b in windows:
            want[i, a] = r.integers(0, 256, b - a, np.uint8)
            for s, x in ((f, want[i, a]), (to[i], np.zeros(b - a, np.uint8))):
                hip.device_memcpy(p.value + int(s) * slot + a, x.ctypes.data, x.nbytes, capi.HOST_TO_DEVICE)
    assert hip.nvllm_copy_states(p, slot, 1, 2 * n, capi.ints(frm), capi.ints(to), n) == 0
    for (i, a), x in want.items():
        for s in (frm[i], to[i]):
            np.testing.assert_array_equal(hip.to_host(p.value + int(s) * slot + a, x.shape, np.uint8), x)
    hip.free(p.value)
