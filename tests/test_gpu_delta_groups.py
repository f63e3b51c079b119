"""More portions than have room for their chunks' records together: they go in groups."""
import pytest

from tests.test_gpu_gated_delta import BOTH, check

pytestmark = pytest.mark.gpu


@BOTH
@pytest.mark.parametrize("singles", [0, 40])
def test_groups_of_portions(hip, elem, singles):
    """64 heads have room for 83 chunks: 170 portions go in three groups, the single tokens with the last one's first launch."""
    n = 170
    spans = [((11 * i) % (n + singles), (i % 3) * 5, 76 + i % 70 if i < n else 1) for i in range(n + singles)]
    check(hip, elem, spans, 16, 64, 8, 16, slots=n + singles + 2)


def test_groups_of_rows_that_are_packed(hip):
    check(hip, 2, [(i, 3 * i, 76 + i % 5) for i in range(90)], 32, 64, 5, 3, slots=91)


@pytest.mark.parametrize("singles", [0, 5])
def test_groups_that_travel_with_the_arguments(hip, singles):
    """Few enough sequences for the launch's arguments, too many heads for one group."""
    n = 40
    check(hip, 2, [(i, i, 76 + 9 * (i % 13) if i < n else 1) for i in range(n + singles)], 60, 240, 8, 8, slots=n + singles)
