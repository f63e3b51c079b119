"""Copies of states and blocks, forked and compacted tables: what lies in HBM afterwards, byte for byte."""
import ctypes as C

import numpy as np
import pytest

from nvllm_amd import capi
from tests import hybrid_util as H
from tests import latent_util as LU

pytestmark = pytest.mark.gpu


def rng(seed):
    return np.random.Generator(np.random.PCG64(seed))


def simultaneous(x, frm, to):
    """[layers, slots, ...] after the copy."""
    y = x.copy()
    y[:, to] = x[:, frm]
    return y


MOVES = {
    "one": ([3], [0]),
    "fan": ([2] * 9, [0, 1, 3, 4, 5, 6, 7, 8, 9]),
    "swap": ([0, 1], [1, 0]),
    "chain": ([0, 1, 2, 3], [1, 2, 3, 4]),
    "chain, last first": ([3, 2, 1, 0], [4, 3, 2, 1]),
    "cycle with branches": ([0, 1, 2, 2, 6, 0], [1, 2, 0, 6, 7, 9]),
    "two cycles, one slot onto itself": ([0, 1, 2, 5, 6, 8], [1, 2, 0, 6, 5, 8]),
    "a fan out of a slot that is written": ([4, 4, 4, 4, 4, 4, 9], [0, 1, 2, 3, 5, 6, 4]),
}


@pytest.mark.parametrize("moves", MOVES.values(), ids=MOVES.keys())
@pytest.mark.parametrize("nbytes", [4096 * 5 + 16, 8192, 16, 1234 * 4, 4, 1027, 1])
def test_states(hip, moves, nbytes):
    """Slots of every alignment; the layers lie behind one another, so slots of odd sizes begin anywhere."""
    frm, to = moves
    x = rng(nbytes).integers(0, 256, (3, 10, nbytes), np.uint8)
    margin = np.full(64, 0xa5, np.uint8)
    p = hip.to_device(np.concatenate([x.reshape(-1), margin]))
    assert hip.nvllm_copy_states(p, nbytes, 3, 10, capi.ints(frm), capi.ints(to), len(to)) == 0
    got = hip.to_host(p, (x.size + 64,), np.uint8)
    np.testing.assert_array_equal(got[:-64].reshape(x.shape), simultaneous(x, frm, to))
    assert (got[-64:] == 0xa5).all()
    hip.free(p)


@pytest.mark.parametrize("seed", range(6))
def test_states_of_many_beams(hip, seed):
    """Every beam's parent is some beam: more moves than travel with a launch's arguments."""
    r = rng(seed)
    slots = 300
    to = r.permutation(slots)[:260]
    frm = to[r.integers(0, 260 if seed % 2 else 4, 260)]
    x = r.integers(0, 256, (2, slots, 48 + 4 * seed), np.uint8)
    p = hip.to_device(x)
    assert hip.nvllm_copy_states(p, x.shape[2], 2, slots, capi.ints(frm), capi.ints(to), 260) == 0
    np.testing.assert_array_equal(hip.to_host(p, x.shape, np.uint8), simultaneous(x, frm, to))
    hip.free(p)


def test_states_behind_the_first_four_gigabytes(hip):
    slots, nbytes = 70, 1 << 26
    p = C.c_void_p()
    assert hip.device_malloc(C.byref(p), slots * nbytes) == 0
    x = rng(1).integers(0, 256, nbytes, np.uint8)
    hip.device_memcpy(p.value + 68 * nbytes, x.ctypes.data, nbytes, capi.HOST_TO_DEVICE)
    assert hip.nvllm_copy_states(p, nbytes, 1, slots, capi.ints([68, 68]), capi.ints([69, 2]), 2) == 0
    for s in (2, 68, 69):
        np.testing.assert_array_equal(hip.to_host(p.value + s * nbytes, (nbytes,), np.uint8), x)
    hip.free(p)


# ------------------------------------------------------------------ pools


class Pool:
    """Any of the library's pools; arrays: (byte offset in keys' or values' memory, bytes of a block) of everything that a block has."""

    def __init__(self, hip, kind, blocks):
        self.hip, self.m, self.n, self.own = hip, capi.KVCacheManager(), blocks, []
        m = C.byref(self.m)
        if kind in ("f32", "f16", "attached"):
            eb, layers, kvh, hd = (2, 3, 2, 48) if kind == "f16" else (4, 3, 2, 40)
            block = 16 * kvh * hd * eb
            if kind == "attached":
                self.own = [hip.empty_device(layers * blocks * block) for _ in range(2)]
                assert hip.nvllm_attach_kv_pool(m, 16, blocks, layers, kvh, hd, eb, *self.own) == 0
            else:
                hip.nvllm_set_kv_elem_bytes(eb)
                hip.init_kv_cache_manager(m, 16, blocks, layers, kvh, hd)
                hip.nvllm_set_kv_elem_bytes(4)
            self.arrays = [(which, i * blocks * block, block) for which in (0, 1) for i in range(layers)]
            self.bytes = [layers * blocks * block] * 2
        elif kind.startswith("latent"):
            eb = int(kind[-1])
            row = 20 + 12 if eb == 4 else 32 + 32
            hip.nvllm_latent_pool_init(m, 16, blocks, 20, 12, eb)
            self.arrays, self.bytes = [(0, 0, 16 * row * eb)], [blocks * 16 * row * eb]
        else:
            eb = int(kind[-1])
            dim, vdim = (22, 13) if eb == 4 else (32, 32)
            hip.nvllm_window_pool_init(m, 32, blocks, 2, 22, 13, eb)
            k, v = 32 * 2 * dim * eb, 32 * 2 * vdim * eb
            self.arrays, self.bytes = [(0, 0, k), (0, blocks * k, v)], [blocks * (k + v)]
        self.bs = self.m.block_size

    def memory(self):
        return [self.m.pool_k, self.m.pool_v][:len(self.bytes)]

    def fill(self, seed):
        self.x = [rng(seed + i).integers(0, 256, n, np.uint8) for i, n in enumerate(self.bytes)]
        for p, x in zip(self.memory(), self.x):
            self.hip.device_memcpy(p, x.ctypes.data, x.nbytes, capi.HOST_TO_DEVICE)

    def copied(self, frm, to):
        """What memory holds after a copy of blocks."""
        y = [x.copy() for x in self.x]
        for which, at, size in self.arrays:
            src = self.x[which][at:at + self.n * size].reshape(self.n, size)
            y[which][at:at + self.n * size].reshape(self.n, size)[to] = src[frm]
        return y

    def check(self, want):
        for p, y in zip(self.memory(), want):
            np.testing.assert_array_equal(self.hip.to_host(p, y.shape, np.uint8), y)
        self.x = want

    def table(self, blocks, room=32):
        at = (C.c_int * room)(*blocks)
        t = capi.BlockTable(C.cast(at, capi.c_int_p), len(blocks))
        t.keep = at
        return t

    def take(self, n):
        return self.table([self.hip.alloc_block(C.byref(self.m)) for _ in range(n)])

    def close(self):
        self.hip.free_kv_cache_manager(C.byref(self.m))
        for p in self.own:
            self.hip.free(p)   # (still the caller's)


def pointers(tables):
    return (C.POINTER(capi.BlockTable) * len(tables))(*[C.pointer(t) for t in tables])


def blocks(t):
    return t.block_indices[:t.num_blocks]


KINDS = pytest.mark.parametrize("kind", ["f32", "f16", "attached", "latent4", "latent2", "window4", "window2"])


@KINDS
def test_blocks(hip, kind):
    p = Pool(hip, kind, 11)
    p.fill(1)
    for frm, to in (([0, 1, 2], [1, 0, 10]), ([4] * 5, [0, 1, 2, 3, 5]), ([7, 8, 9, 10], [8, 9, 10, 7])):
        want = p.copied(frm, to)
        assert hip.nvllm_copy_blocks(C.byref(p.m), capi.ints(frm), capi.ints(to), len(to)) == 0
        p.check(want)
    p.close()


@KINDS
def test_forks(hip, kind):
    p = Pool(hip, kind, 14)
    p.fill(2)
    t = p.take(3)
    to = [p.table([]) for _ in range(5)]
    positions = 2 * p.bs + 1
    want = p.copied([2] * 5, [3, 4, 5, 6, 7])
    assert hip.nvllm_fork_tables(C.byref(p.m), C.byref(t), positions, pointers(to), 5) == 0
    assert [blocks(x) for x in to] == [[0, 1, 3 + i] for i in range(5)]
    p.check(want)
    # a branch branches at a block's end: nothing is copied
    more = [p.table([])]
    assert hip.nvllm_fork_tables(C.byref(p.m), C.byref(to[3]), 2 * p.bs, pointers(more), 1) == 0 and blocks(more[0]) == [0, 1]
    p.check(want)
    assert [hip.nvllm_block_users(C.byref(p.m), b) for b in range(9)] == [7, 7, 1, 1, 1, 1, 1, 1, 0]
    p.close()


@KINDS
def test_compaction(hip, kind):
    p = Pool(hip, kind, 16)
    p.fill(3)
    m = C.byref(p.m)
    a, b, c = p.take(4), p.take(4), p.take(4)                      # 0-3, 4-7, 8-11
    forked = [p.table([])]
    assert hip.nvllm_fork_tables(m, C.byref(c), 3 * p.bs, pointers(forked), 1) == 0
    assert hip.nvllm_free_table(m, C.byref(a)) == 0                # 4-11 in use
    want = p.copied([8, 9, 10, 11], [0, 1, 2, 3])
    assert hip.nvllm_compact_blocks(m, pointers([b, c, forked[0]]), 3) == 4
    assert (blocks(b), blocks(c), blocks(forked[0])) == ([4, 5, 6, 7], [0, 1, 2, 3], [0, 1, 2])
    p.check(want)
    assert [hip.nvllm_block_users(m, i) for i in range(9)] == [2, 2, 2, 1, 1, 1, 1, 1, 0]
    assert p.m.free_block_indices[:p.m.free_blocks_count] == list(range(15, 7, -1))
    assert hip.nvllm_compact_blocks(m, pointers([b, c, forked[0]]), 3) == 0
    p.check(want)
    # every user frees its table: all blocks come back
    for t in (c, b, forked[0]):
        assert hip.nvllm_free_table(m, C.byref(t)) == 0
    assert sorted(p.m.free_block_indices[:16]) == list(range(16))
    p.close()


def test_compaction_around_a_block_that_no_table_has(hip):
    p = Pool(hip, "f32", 12)
    p.fill(4)
    a, b = p.take(5), p.take(5)
    for i in (1, 3):
        hip.free_block(C.byref(p.m), blocks(a)[i])
    rest = p.table([0, 2, 4])
    keep = blocks(b)[1:]          # 6-9; block 5 is somebody else's
    t = p.table(keep)
    want = p.copied([8, 9], [1, 3])
    assert hip.nvllm_compact_blocks(C.byref(p.m), pointers([rest, t]), 2) == 2
    assert (blocks(rest), blocks(t)) == ([0, 2, 4], [6, 7, 1, 3])
    p.check(want)
    assert p.m.free_block_indices[:p.m.free_blocks_count] == [11, 10, 9, 8]
    p.close()


# ------------------------------------------------------------------ a hybrid sequence branches


class Runner:
    """A model folder's passes with tables of the test's own."""

    def __init__(self, hip, path, f32):
        self.hip = hip
        hip.nvllm_set_compute_dtype(capi.COMPUTE_F32 if f32 else capi.COMPUTE_BF16)
        hip.nvllm_set_logits_mode(0)
        self.cfg, self.w, self.s, self.m = capi.Config(), capi.Weights(), capi.RunState(), capi.KVCacheManager()
        hip.load_model(C.byref(self.w), C.byref(self.cfg), path.encode())
        self.cfg.max_seq_len = 512
        hip.malloc_run_state(C.byref(self.s), C.byref(self.cfg))
        hip.nvllm_init_model_kv(C.byref(self.m), 16, 60, C.byref(self.cfg), C.byref(self.w))
        hip.nvllm_init_model_states(C.byref(self.w), 6)
        self.tables = {}

    def run(self, parts):
        """parts: (sequence, first position, tokens); the last token's logits of each."""
        for i, at, t in parts:
            if i not in self.tables:
                arr = (C.c_int * 40)()
                self.tables[i] = capi.BlockTable(C.cast(arr, capi.c_int_p), 0)
                self.tables[i].keep = arr
            table = self.tables[i]
            while table.num_blocks * 16 < at + len(t):
                table.block_indices[table.num_blocks] = self.hip.alloc_block(C.byref(self.m))
                table.num_blocks += 1
        ptrs = (C.POINTER(capi.BlockTable) * 6)(*[C.pointer(self.tables[i]) if i in self.tables else None for i in range(6)])
        C.memmove(C.addressof(capi.KVCacheManager.in_dll(self.hip.dll, "g_kv_manager")), C.addressof(self.m), C.sizeof(self.m))
        toks = capi.ints(np.concatenate([t for _, _, t in parts]))
        pos = capi.ints(np.concatenate([np.arange(at, at + len(t)) for _, at, t in parts]))
        ids = capi.ints(np.concatenate([np.full(len(t), i) for i, _, t in parts]))
        out = capi.ints(np.cumsum([len(t) for _, _, t in parts]) - 1)
        self.hip.transformer_batch(toks, len(toks), pos, ids, out, len(parts), C.byref(self.cfg), C.byref(self.s), C.byref(self.w), ptrs)
        return np.ctypeslib.as_array(C.cast(self.s.logits, capi.c_float_p), shape=(len(parts), self.cfg.vocab_size)).copy()

    def close(self):
        self.hip.free_kv_cache_manager(C.byref(self.m))
        self.hip.free_run_state(C.byref(self.s))
        self.hip.nvllm_free_model(C.byref(self.w))


@pytest.mark.parametrize("f32", [True, False], ids=["fp32", "bf16"])
@pytest.mark.parametrize("design", ["simivik odd", "simivik parts", "suselorn odd"])
def test_branches_go_on_like_the_sequence_itself(hip, tmp_path, design, f32):
    """A sequence of 37 positions branches twice; sequence and branches take tokens of their own; the pool is compacted in between.
    Their logits are those of sequences that were fed everything from the start."""
    family, name = design.split()
    path, cfg, _ = (H if family == "simivik" else LU).model(tmp_path, name)
    r = Runner(hip, path, f32)
    prompt = LU.tokens(37, cfg["vocab"], 1)
    tails = [LU.tokens(n, cfg["vocab"], 5 + n) for n in (12, 9, 1)]
    want = [r.run([(5, 0, np.concatenate([prompt, t]))])[0] for t in tails]
    assert hip.nvllm_free_table(C.byref(r.m), C.byref(r.tables.pop(5))) == 0
    hold = [hip.alloc_block(C.byref(r.m)) for _ in range(7)]   # what the pool's front is taken by
    r.run([(0, 0, prompt)])
    branches = []
    for _ in range(2):
        arr = (C.c_int * 40)()
        branches.append(capi.BlockTable(C.cast(arr, capi.c_int_p), 0))
        branches[-1].keep = arr
    assert hip.nvllm_fork_tables(C.byref(r.m), C.byref(r.tables[0]), 37, pointers(branches), 2) == 0
    assert hip.nvllm_copy_model_states(C.byref(r.w), capi.ints([0, 0]), capi.ints([2, 3]), 2) == 0
    r.tables[2], r.tables[3] = branches
    r.run([(2, 37, tails[1][:4]), (0, 37, tails[0][:5])])
    for b in hold:
        hip.free_block(C.byref(r.m), b)
    assert hip.nvllm_compact_blocks(C.byref(r.m), pointers([r.tables[i] for i in (0, 2, 3)]), 3) > 0
    got = r.run([(0, 42, tails[0][5:]), (3, 37, tails[2]), (2, 41, tails[1][4:])])
    for i, w in zip((0, 2, 1), want):
        assert LU.error(got[i:i + 1], w[None]) < LU.limit(f32)
    assert hip.nvllm_copy_model_states(C.byref(r.w), capi.ints([0]), capi.ints([6]), 1) == (0 if family == "suselorn" else -3)
    r.close()


def test_a_model_file_keeps_no_states(hip, tmp_models):
    path, _ = tmp_models("tiny")
    w, cfg = capi.Weights(), capi.Config()
    hip.load_model(C.byref(w), C.byref(cfg), path.encode())
    assert hip.nvllm_copy_model_states(C.byref(w), capi.ints([0]), capi.ints([1]), 1) == 0
    assert hip.nvllm_copy_model_states(None, capi.ints([0]), capi.ints([1]), 1) == -1
    assert hip.nvllm_copy_model_states(C.byref(w), None, capi.ints([1]), 1) == -1
    hip.nvllm_free_model(C.byref(w))
