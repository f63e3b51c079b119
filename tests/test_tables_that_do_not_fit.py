"""Tables that name a block twice or one that is free: refused as a whole, without a GPU."""
import ctypes as C

import pytest

from tests.test_sequence_memory import BAD_INDEX, Pool, blocks, lib  # noqa: F401


@pytest.mark.parametrize("wrong", [[3, 3], [0, 3, 0], [3, 9], [9], [4, 3, 12], [-1, 3]], ids=str)
def test_releases_that_are_refused_change_nothing(lib, wrong):  # noqa: F811
    p = Pool(lib)
    p.take(5)
    t = p.take(2)
    rc, (child,) = p.fork(t, 32, 1)
    stack = p.stack()
    bad = p.table(wrong)
    assert rc == 0 and p.free(bad) == BAD_INDEX
    assert blocks(bad) == wrong and p.stack() == stack and [p.users(i) for i in range(8)] == [1] * 5 + [2, 2, 0]
    shared = p.table([5, 6, 5])
    assert p.free(shared) == BAD_INDEX and blocks(shared) == [5, 6, 5] and [p.users(i) for i in (5, 6)] == [2, 2]
    assert p.free(child) == 0 and p.free(t) == 0 and p.stack() == stack + [6, 5]
    again = p.table([5])
    assert p.free(again) == BAD_INDEX and p.stack() == stack + [6, 5]


@pytest.mark.parametrize("count", [-1, 5, 6, 7])
def test_a_stack_without_room(lib, count):  # noqa: F811
    """A stack that says it holds more than the blocks which nobody uses."""
    p = Pool(lib, 6)
    t = p.take(2)
    p.m.free_blocks_count = count
    assert p.free(t) == BAD_INDEX and blocks(t) == [0, 1] and p.m.free_blocks_count == count


def test_a_stack_with_a_number_that_is_no_block(lib):  # noqa: F811
    p = Pool(lib, 6)
    t = p.take(2)
    for bad in (6, -1, 1 << 30):
        p.m.free_block_indices[1] = bad
        assert p.free(t) == BAD_INDEX and blocks(t) == [0, 1] and p.m.free_blocks_count == 4
    p.m.free_block_indices[1] = 4
    assert p.free(t) == 0 and p.m.free_blocks_count == 6


def test_every_block_of_a_pool_comes_back_once(lib):  # noqa: F811
    p = Pool(lib, 40)
    tables = [p.take(n) for n in (1, 0, 7, 16, 16)]
    assert p.m.free_blocks_count == 0
    for t in tables:
        assert p.free(t) == 0
        assert p.free(t) == 0   # (empty by now)
    assert sorted(p.stack()) == list(range(40))
    assert lib_users(p) == [0] * 40


def lib_users(p):
    return [p.lib.nvllm_block_users(C.byref(p.m), b) for b in range(p.m.num_blocks)]
