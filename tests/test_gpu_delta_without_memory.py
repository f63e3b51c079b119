"""A call whose workspace is larger than the GPU: refused by the runtime itself, and the next call goes on."""
import numpy as np
import pytest

from nvllm_amd import capi
from tests.test_gpu_gated_delta import BOTH, Buffers, check

pytestmark = pytest.mark.gpu


@BOTH
def test_rows_that_do_not_fit_when_packed(hip, elem):
    """65,535 heads of one dim: a row to pack takes eight times its bytes, three terabytes of 16 bits in all.  Nothing is enqueued, so nothing reads
    or writes the buffers, which are far smaller than the call says."""
    T, H = 1_000_000, 65535
    b = Buffers(hip)
    mark = np.arange(64, dtype=np.float32)
    p = [b.put(mark) for _ in range(7)]
    ids = np.zeros(T, np.int32).ctypes.data_as(capi.c_int_p)
    pos = np.arange(T, dtype=np.int32).ctypes.data_as(capi.c_int_p)
    assert hip.nvllm_gated_delta(*p, ids, pos, 1, 1.0, 0.0, H, H, 1, 1, H, H, H, elem, T) == -5
    hip.device_sync()
    for x in p:
        np.testing.assert_array_equal(b.get(x, mark.shape, np.float32), mark)
    b.free()
    check(hip, elem, [(0, 3, 100), (1, 0, 1)], 2, 2, 40, 24)
