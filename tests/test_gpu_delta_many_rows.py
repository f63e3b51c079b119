"""More rows to pack than workgroups that pack them: the results are those of rows that need no packing, to the bit."""
import numpy as np
import pytest

from tests import delta_oracle as O
from tests.test_gpu_gated_delta import BOTH, call

pytestmark = pytest.mark.gpu


@BOTH
def test_a_million_rows(hip, elem):
    T = (1 << 20) + 300
    data = O.inputs(5, T, 1, 1, 8, 8, elem, 2)
    spans = [(1, 0, T - 100), (0, 7, 100)]
    aligned = call(hip, data, spans, elem, 0.5, 1e-6)
    packed = call(hip, data, spans, elem, 0.5, 1e-6, extra=3, shift=elem)
    for a, b in zip(aligned, packed):
        np.testing.assert_array_equal(a, b)
    assert np.isfinite(aligned[0]).all()
