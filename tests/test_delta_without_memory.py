"""Calls whose workspace finds no memory are refused before anything is enqueued or changed; a stand-in takes the runtime's place."""
from tests import hip_standin

NO_MEMORY = -5
CALLS = """
def refused(call):
    gpu.standin_forget()
    assert call() == -5
    assert gpu.standin_launches() == 0, launches()
def passes(call):
    gpu.standin_forget()
    assert call() == 0 and gpu.standin_launches() > 0
"""


def test_records_of_chunks(tmp_path):
    hip_standin.run(tmp_path, CALLS + """
ids, pos = np.repeat(np.arange(3), 700), np.tile(np.arange(700), 3)
call = lambda: delta(ids, pos, 3, 16, 64, 64)
gpu.standin_memory(4 << 20)
refused(call)
refused(lambda: delta(ids, pos, 3, 16, 5, 7, q_ld=83))   # rows that would be packed
gpu.standin_memory(1 << 30)
passes(call)
""")


def test_more_sequences_than_travel_with_a_launch(tmp_path):
    hip_standin.run(tmp_path, CALLS + """
n = 5000
one = lambda: delta(np.arange(n), np.full(n, 3), n, 2, 32, 32)
some = lambda: delta(np.repeat(np.arange(200), 100), np.tile(np.arange(100), 200), 200, 2, 32, 32)
gpu.standin_memory(1000)
refused(one)
refused(some)
gpu.standin_memory(1 << 20)      # room for the sequences, not for the records
refused(some)
passes(one)
gpu.standin_memory(1 << 30)
passes(some)
passes(one)
""")
