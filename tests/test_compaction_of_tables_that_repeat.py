"""Compaction counts the tables that have a block: a table that names one twice is one table.  Nothing moves here."""
from tests.test_sequence_memory import Pool, blocks, lib  # noqa: F401


def test_a_table_that_names_a_block_twice(lib):  # noqa: F811
    p = Pool(lib, 8)
    a, b = p.take(2), p.take(2)
    rc, (c,) = p.fork(b, 32, 1)                      # 2 and 3: two users each
    assert rc == 0 and p.free(a) == 0
    twice = p.table([2, 3, 2, 3])                    # one of the two users; the other one's table is not given
    assert p.compact([twice]) == 0
    assert p.stack() == [7, 6, 5, 4, 1, 0] and blocks(twice) == [2, 3, 2, 3] and blocks(b) == blocks(c) == [2, 3] and [p.users(i) for i in range(4)] == [0, 0, 2, 2]
