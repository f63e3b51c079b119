"""Launches of more workgroups than a grid takes (2^32 threads): a stand-in takes the runtime's place and refuses them as the runtime does."""
import pytest

from tests import hip_standin

CHECK = """
def fits():
    assert gpu.standin_launches() > 0
    for g, b in launches():
        assert g[0] * b[0] < 1 << 32 and g[1] < 65536 and g[2] < 65536, (g, b)
"""


@pytest.mark.parametrize("slot,n", [((1 << 31) - 1, 8), ((1 << 30) + 1, 40), (4 * ((1 << 30) + 1), 9), (16 << 29, 9), (1, 200000), (8193 * 16, 200000)], ids=str)
def test_copies(tmp_path, slot, n):
    """Slots of odd sizes (a byte a thread) and of whole vectors; few moves of large slots, many of small ones."""
    hip_standin.run(tmp_path, CHECK + """
slot, n = %d, %d
assert lib.nvllm_copy_states(0x100000000000, slot, 2, 2 * n, ints(np.arange(n)), ints(np.arange(n) + n), n) == 0
fits()
unit = 16 if slot %% 16 == 0 else 4 if slot %% 4 == 0 else 1
work = [g for g, b in launches() if g[1] == 2]
assert sum(g[0] for g in work) == n * -(-slot // unit // 512)   # every piece of every move once
""" % (slot, n))


@pytest.mark.parametrize("tokens", [1 << 24, (1 << 24) + 5], ids=str)
def test_packed_rows(tmp_path, tokens):
    """A portion of 16 million tokens whose rows are packed, a workgroup a row."""
    hip_standin.run(tmp_path, CHECK + """
n = %d
assert delta(np.zeros(n), np.arange(n), 1, 1, 5, 3) == 0
fits()
""" % tokens)
