"""The largest strides and widths that nvllm_gated_delta takes: a chunk's last row begins 2^31 bytes behind its first, less a row."""
import ctypes as C

import numpy as np
import pytest

from nvllm_amd import capi
from tests import delta_oracle as O
from tests.test_gpu_gated_delta import BOTH, Buffers, stored

pytestmark = pytest.mark.gpu
MOST = 1 << 23


@BOTH
@pytest.mark.parametrize("n", [70, 9], ids=["chunks", "token by token"])
@pytest.mark.parametrize("ld", [MOST, MOST - 1], ids=["aligned", "odd"])
def test_rows_far_apart(hip, elem, n, ld):
    """q, k and v are parts of one row of 2^23 elements: at its start, in its middle and at its end."""
    Q, H, dim, vdim = 1, 2, 40, 24
    data = O.inputs(n + elem, n, Q, H, dim, vdim, elem, 2)
    q, k, v, g, beta, state = data
    base = C.c_void_p()
    assert hip.device_malloc(C.byref(base), n * ld * elem) == 0
    first = [0, (ld // 2) & ~7, (ld - H * vdim) & ~7]
    for t in range(n):
        for x, at in zip((q, k, v), first):
            row = stored(x[t], elem).reshape(-1)
            hip.device_memcpy(base.value + (t * ld + at) * elem, row.ctypes.data, row.nbytes, capi.HOST_TO_DEVICE)
    b = Buffers(hip)
    out, ds, dg, db = b.put(stored(np.full(v.shape, np.nan, np.float32), elem)), b.put(state), b.put(g), b.put(beta)
    rc = hip.nvllm_gated_delta(out, *(base.value + at * elem for at in first), dg, db, ds, capi.ints([1] * n), capi.ints(range(5, 5 + n)), 2, 0.25, 1e-6, Q, H, dim, vdim, ld, ld, ld, elem, n)
    assert rc == 0
    got = b.get(out, v.shape, np.uint16 if elem == O.BF16 else np.float32)
    got, st = O.from_bf16(got) if elem == O.BF16 else got, b.get(ds, state.shape, np.float32)
    b.free()
    hip.free(base.value)
    want, wanted = O.forward(*data, [(1, 5, n)], np.float32(0.25), 1e-6)
    assert O.off(got, want, elem) <= O.limit(n, dim) and O.off(st[1:], wanted[1:]) <= O.limit(n, dim)
    np.testing.assert_array_equal(st[0], state[0])


@BOTH
def test_the_widest_results(hip, elem):
    """heads * vdim at its limit: 2^23 values a token, of 128 heads, whose columns are alike in threes."""
    n, H, vdim, dim = 66, 128, 1 << 16, 8
    vdim -= 16                                     # (65,535 columns at most; a multiple of 16 that is not one of 32)
    r = O.inputs(3, n, 1, 1, dim, 3, elem, 1)
    q, k, v3, g1, b1, _ = r
    dq, dk, dg, db = Buffers(hip), Buffers(hip), np.repeat(g1, H, 1), np.repeat(b1, H, 1)
    pq, pk = dq.put(stored(q, elem)), dk.put(stored(k, elem))
    row = np.resize(np.arange(3), vdim)
    one = stored(v3[:, 0][:, row], elem)           # [n, vdim], the same for every head
    size = n * H * vdim * elem
    pv, po, ps = C.c_void_p(), C.c_void_p(), C.c_void_p()
    for p, bytes_ in ((pv, size), (po, size + 256), (ps, H * dim * vdim * 4)):
        assert hip.device_malloc(C.byref(p), bytes_) == 0
    for t in range(n):
        x = np.tile(one[t], H)
        hip.device_memcpy(pv.value + t * H * vdim * elem, x.ctypes.data, x.nbytes, capi.HOST_TO_DEVICE)
    mark = np.full(256, 0xa5, np.uint8)
    hip.device_memcpy(po.value + size, mark.ctypes.data, 256, capi.HOST_TO_DEVICE)
    pg, pb = dq.put(dg), dk.put(db)
    ld = H * vdim
    assert hip.nvllm_gated_delta(po.value, pq, pk, pv.value, pg, pb, ps.value, capi.ints([0] * n), capi.ints(range(n)), 1, 0.5, 1e-6, 1, H, dim, vdim, dim, dim, ld, elem, n) == 0
    want, wanted = O.forward(q, k, v3, g1, b1, np.zeros((1, 1, dim, 3), np.float32), [(0, 0, n)], np.float32(0.5), 1e-6)
    most = O.limit(n, dim)
    for t in (0, 1, 40, 63, 64, n - 1):
        for h in (0, 77, H - 1):
            got = hip.to_host(po.value + (t * H + h) * vdim * elem, (vdim,), np.uint16 if elem == O.BF16 else np.float32)
            got = O.from_bf16(got) if elem == O.BF16 else got
            rms = np.sqrt((want ** 2).mean())
            d = np.abs(got - want[t, 0][row]) - (2.0 ** -8 * np.abs(want[t, 0][row]) if elem == O.BF16 else 0)
            assert d.max() <= most * rms, (t, h)
    for h in (0, H - 1):
        st = hip.to_host(ps.value + h * dim * vdim * 4, (dim, vdim), np.float32)
        assert np.abs(st - wanted[0, 0][:, row]).max() <= most * np.sqrt((wanted ** 2).mean())
    np.testing.assert_array_equal(hip.to_host(po.value + size, (256,), np.uint8), mark)
    for p in (pv, po, ps):
        hip.free(p.value)
    dq.free()
    dk.free()
