"""Long portions in segments beside more sequences than travel with a launch's arguments: the segments' numbers go further than the sequences'."""
import pytest

from tests.test_gpu_gated_delta import BOTH, check

pytestmark = pytest.mark.gpu


@BOTH
@pytest.mark.parametrize("long,short", [(64, 33), (30, 70)], ids=str)
def test_segments_of_many_sequences(hip, elem, long, short):
    """One head, so that 64 portions of 30 chunks go in three segments each."""
    check(hip, elem, [(i, 3 * i, 1900 - i if i < long else 1) for i in range(long + short)], 1, 1, 32, 16)
