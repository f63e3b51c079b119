"""What nvllm_gated_delta asks of the GPU's memory and launches; a stand-in takes the runtime's place, no kernel runs."""
import pytest

from tests import hip_standin

RECORDS = 192 << 20   # bytes of the chunks' records of a launch
HEADROOM = 1.26       # of a workspace that grows


@pytest.mark.parametrize("n,per,heads", [(2048, 80, 64), (300, 700, 64), (70000, 80, 1), (5, 4000, 4096), (3, 20000, 16)], ids=str)
def test_records_stay_within_their_room(tmp_path, n, per, heads):
    """However many portions a batch has; a portion whose one chunk has more gets that much."""
    hip_standin.run(tmp_path, """
n, per, heads = %d, %d, %d
assert delta(np.repeat(np.arange(n), per), np.tile(np.arange(per), n), n, heads, 32, 16) == 0
most = max(%d, heads * 37888)
assert gpu.standin_largest() <= %g * most, gpu.standin_largest()
work = [g for g, b in launches() if b[0] == 512]   # the walks: every chunk of every portion once
assert all(g[2] <= 65535 for g in work) and sum(g[2] for g in work) >= n
""" % (n, per, heads, RECORDS, HEADROOM))
