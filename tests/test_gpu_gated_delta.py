"""The gated delta rule through its entry point against its definition in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from nvllm_amd import capi
from tests import delta_oracle as O

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("elem", [O.F32, O.BF16], ids=["fp32", "bf16"])


class Buffers:
    """Device buffers of a test, guarded by a margin of known bytes behind each."""
    MARGIN = 256

    def __init__(self, hip):
        self.hip, self.all = hip, []

    def put(self, arr, shift=0):
        """shift: bytes that the array lies behind a multiple of 256."""
        raw = np.frombuffer(np.ascontiguousarray(arr).tobytes(), np.uint8)
        buf = np.full(shift + raw.size + self.MARGIN, 0xa5, np.uint8)
        buf[shift:shift + raw.size] = raw
        p = self.hip.to_device(buf)
        self.all.append((p, shift, raw.size))
        return p + shift

    def get(self, ptr, shape, dtype):
        p, shift, n = next(b for b in self.all if b[0] + b[1] == ptr)
        buf = self.hip.to_host(p, (shift + n + self.MARGIN,), np.uint8)
        assert (buf[:shift] == 0xa5).all() and (buf[shift + n:] == 0xa5).all(), "written beside a buffer"
        return buf[shift:shift + n].copy().view(dtype).reshape(shape)

    def free(self):
        for p, _, _ in self.all:
            self.hip.free(p)


def stored(x, elem):
    return O.to_bf16(x) if elem == O.BF16 else np.ascontiguousarray(x, np.float32)


def rows(parts, elem, extra):
    """Heads of a token side by side, `extra` elements of rubbish behind each row; returns the array and its row length."""
    flat = np.concatenate([stored(p, elem).reshape(len(p), -1) for p in parts], 1)
    junk = stored(np.full((len(flat), extra), np.nan, np.float32), elem)
    a = np.concatenate([flat, junk], 1)
    return a, a.shape[1]


def call(hip, data, spans, elem, scale, eps, fused=False, extra=0, shift=0, state=None):
    q, k, v, g, beta, st = data
    st = st if state is None else state
    T, Q, dim = q.shape
    H, vdim = v.shape[1:]
    b = Buffers(hip)
    size = elem
    if fused:
        a, ld = rows([q, k, v], elem, extra)
        base = b.put(a, shift)
        ptrs, lds = (base, base + Q * dim * size, base + 2 * Q * dim * size), (ld, ld, ld)
    else:
        made = [rows([x], elem, extra) for x in (q, k, v)]
        ptrs, lds = [b.put(a, shift) for a, _ in made], [ld for _, ld in made]
    out = b.put(stored(np.full(v.shape, np.nan, np.float32), elem), shift)
    ds, dg, db = b.put(st), b.put(g), b.put(beta)
    ids = capi.ints([s for s, _, n in spans for _ in range(n)])
    pos = capi.ints([p + i for _, p, n in spans for i in range(n)])
    rc = hip.nvllm_gated_delta(out, *ptrs, dg, db, ds, ids, pos, len(st), scale, eps, Q, H, dim, vdim, *lds, elem, T)
    assert rc == 0
    o = b.get(out, v.shape, np.uint16 if elem == O.BF16 else np.float32)
    s = b.get(ds, st.shape, np.float32)
    b.free()
    return (O.from_bf16(o) if elem == O.BF16 else o), s


def check(hip, elem, spans, Q, H, dim, vdim, slots=None, eps=1e-6, seed=0, unit_keys=False, scale=None, edit=None, **kw):
    T, slots = sum(n for _, _, n in spans), slots or max(s for s, _, _ in spans) + 2
    data = O.inputs(seed + 7 * T + dim, T, Q, H, dim, vdim, elem, slots, unit_keys)
    if edit:
        edit(*data)
    scale = np.float32(dim ** -0.5 if scale is None else scale)
    got, state = call(hip, data, spans, elem, scale, eps, **kw)
    want, wanted = O.forward(*data, spans, scale, eps)
    most = O.limit(max(n for _, _, n in spans), dim)
    used = [s for s, _, _ in spans]
    worst = O.off(got, want, elem), O.off(state[used], wanted[used])
    assert worst[0] <= most and worst[1] <= most, (worst, most)
    rest = [s for s in range(slots) if s not in used]
    np.testing.assert_array_equal(state[rest], data[5][rest])
    return got, state


# one head, heads that share queries and keys; dims of every register count, off every vector width; columns that end inside a wave's
HEADS = [(1, 1, 64, 64), (2, 6, 32, 32), (4, 4, 128, 128), (1, 2, 40, 100), (2, 2, 96, 48), (1, 3, 192, 24), (1, 1, 256, 256), (2, 2, 57, 33), (3, 3, 1, 1), (1, 1, 250, 5)]


@BOTH
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_single_tokens(hip, elem, heads):
    check(hip, elem, [(3, 17, 1), (0, 0, 1), (5, 1, 1), (1, 900, 1)], *heads)


@BOTH
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_portions_of_unlike_lengths(hip, elem, heads):
    check(hip, elem, [(2, 0, 5), (0, 63, 2), (4, 8, 1), (3, 0, 70), (1, 64, 131)], *heads)


@BOTH
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 79, 127, 128, 129, 191, 192, 193, 257, 640])
def test_lengths(hip, elem, n):
    check(hip, elem, [(1, 0, n)], 2, 4, 64, 64)
    check(hip, elem, [(0, 5, n)], 1, 1, 128, 96, unit_keys=True, eps=0.0)


@BOTH
def test_a_long_portion(hip, elem):
    check(hip, elem, [(0, 3, 2500)], 1, 2, 128, 64)


@BOTH
@pytest.mark.parametrize("n", [6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 22, 23, 28, 29, 33, 34, 42, 43])
def test_short_portions(hip, elem, n):
    """About the lengths at which chunks take over, which rise with the batch."""
    check(hip, elem, [(1, 0, n), (0, 60, n + 1)], 2, 2, 64, 48)
    check(hip, elem, [(i, 3 * i, n + i % 2) for i in range(8)], 16, 32, 32, 128)


# few heads and many tokens: such portions are walked in segments side by side; heads of every number of 32 dims, columns off every width
LONG = [(1, 2, 32, 20, 900), (1, 1, 64, 64, 1500), (1, 3, 80, 16, 1300), (2, 2, 128, 40, 1700), (1, 1, 192, 24, 2400), (1, 1, 256, 33, 3200)]


@BOTH
@pytest.mark.parametrize("heads", LONG, ids=str)
def test_long_portions_of_few_heads(hip, elem, heads):
    """Beside portions of a chunk, of half the length and of a token."""
    *heads, n = heads
    check(hip, elem, [(2, 0, n)], *heads)
    check(hip, elem, [(2, 9, n), (0, 70, 50), (1, 5, 1), (5, 0, n // 2 + 3), (3, 0, 65)], *heads, seed=1)


@BOTH
def test_gates_of_long_portions(hip, elem):
    """Heads that hold what they read over the whole portion, that lose all of it in the middle, that never write; a slot of rubbish."""
    def gates(q, k, v, g, beta, state):
        g[:, 0], beta[:, 0] = 0.0, 0.01
        g[700, 1] = -np.inf
        beta[:, 2] = 0.0
        g[:, 2] = -1e-4
        g[:, 3] = -60.0
        state[1] = np.nan
    check(hip, elem, [(0, 9, 1600), (1, 0, 1100)], 2, 4, 64, 32, edit=gates)


@pytest.mark.parametrize("heads", [(16, 16, 32, 16, 40000), (256, 256, 32, 16, 2400)], ids=str)
def test_more_chunks_than_are_prepared_at_a_time(hip, heads):
    """With segments (16 heads) and without; the state goes on from one round of chunks to the next."""
    *heads, n = heads
    check(hip, O.BF16, [(0, 3, n), (1, 0, 100)], *heads)


@BOTH
def test_many_sequences(hip, elem):
    """More portions than travel with a launch's arguments, slots in no order."""
    order = np.random.Generator(np.random.PCG64(5)).permutation(90)
    check(hip, elem, [(int(s), 3 * i, 1 + (i % 3 == 0) * i) for i, s in enumerate(order[:75])], 2, 2, 32, 40, slots=90)


@BOTH
@pytest.mark.parametrize("extra,shift", [(0, 0), (8, 16), (4, 8), (1, 0), (3, 4), (5, 12)], ids=str)
@pytest.mark.parametrize("n", [1, 150])
def test_rows_of_a_fused_projection(hip, elem, extra, shift, n):
    """q, k and v side by side, rows and addresses at every distance from a vector's; what lies behind the rows is not read."""
    check(hip, elem, [(1, 4, n)], 2, 4, 64, 32, fused=True, extra=extra, shift=shift)


@BOTH
@pytest.mark.parametrize("n", [1, 100])
def test_a_portion_starts_from_an_empty_state(hip, elem, n):
    """At position 0 what the slot held does not count, not even what is not a number."""
    def dirty(q, k, v, g, beta, state):
        state[1] = np.nan
    check(hip, elem, [(1, 0, n)], 2, 2, 64, 64, edit=dirty)


@BOTH
def test_edges_of_gates(hip, elem):
    """Heads that never forget and always overwrite; that empty the state at a token; that never write; decays near one and near zero."""
    def gates(q, k, v, g, beta, state):
        g[:, 0], beta[:, 0] = 0.0, 1.0
        g[40::50, 1] = -np.inf
        beta[:, 2] = 0.0
        g[:, 3] = -1e-6
        g[:, 4] = -60.0
        g[7:60, 5] = -200.0
    for n in (1, 45, 200):
        check(hip, elem, [(0, 9, n)], 6, 6, 64, 64, edit=gates)


@BOTH
def test_a_key_that_comes_again(hip, elem):
    """The same key token after token: the state holds one value for it, the last, whatever the number of tokens."""
    def same(q, k, v, g, beta, state):
        k[:] = k[:1]
        g[:] = 0.0
        beta[:] = 1.0
    check(hip, elem, [(0, 0, 200)], 1, 2, 64, 64, edit=same)
    check(hip, elem, [(0, 0, 64)], 1, 1, 128, 32, edit=same, eps=0.0, unit_keys=True)


@BOTH
def test_queries_and_keys_of_zeros(hip, elem):
    def zeros(q, k, v, g, beta, state):
        k[3:9], q[5:20] = 0.0, 0.0
    check(hip, elem, [(0, 2, 80)], 2, 2, 64, 64, edit=zeros)


@BOTH
@pytest.mark.parametrize("size", [1e-8, 1e6])
def test_sizes_of_values(hip, elem, size):
    """Nothing hangs on the scale of values and states."""
    def scaled(q, k, v, g, beta, state):
        v *= np.float32(size)
        state *= np.float32(size)
        if elem == O.BF16:
            v[:] = O.from_bf16(O.to_bf16(v))
    check(hip, elem, [(0, 2, 100), (1, 0, 1)], 2, 2, 64, 64, edit=scaled)


@BOTH
def test_portions_one_after_the_other(hip, elem):
    """A sequence in one call, in portions and token by token: the same results to rounding, the state handed on."""
    T, Q, H, dim, vdim = 300, 2, 4, 64, 64
    data = O.inputs(3, T, Q, H, dim, vdim, elem, 2)
    scale = np.float32(0.125)
    want, wanted = O.forward(*data, [(1, 0, T)], scale, 1e-6)
    for cuts in ([0, T], [0, 64, 128, T], [0, 1, 7, 100, 163, 299, T], [0] + list(range(250, T + 1))):
        state, outs = data[5], []
        for a, b in zip(cuts, cuts[1:]):
            part = tuple(x[a:b] for x in data[:5]) + (state,)
            o, state = call(hip, part, [(1, a, b - a)], elem, scale, 1e-6)
            outs.append(o)
        worst = O.off(np.concatenate(outs), want, elem), O.off(state[1:], wanted[1:])
        assert max(worst) <= O.limit(T, dim), worst


@BOTH
def test_the_same_call_twice_gives_the_same_bits(hip, elem):
    data = O.inputs(11, 700, 4, 4, 128, 128, elem, 3)
    spans = [(2, 0, 500), (0, 70, 130), (1, 3, 70)]
    a, b = (call(hip, data, spans, elem, 0.1, 1e-6) for _ in range(2))
    np.testing.assert_array_equal(a[0], b[0])
    np.testing.assert_array_equal(a[1], b[1])


@BOTH
def test_a_long_portion_twice_gives_the_same_bits(hip, elem):
    data = O.inputs(12, 1700, 1, 2, 128, 128, elem, 3)
    spans = [(2, 0, 1600), (0, 70, 100)]
    a, b = (call(hip, data, spans, elem, 0.1, 1e-6) for _ in range(2))
    np.testing.assert_array_equal(a[0], b[0])
    np.testing.assert_array_equal(a[1], b[1])


@BOTH
@pytest.mark.parametrize("heads", [(2, 2, 32, 40), (2, 4, 64, 64)], ids=str)
def test_portions_beside_single_tokens(hip, elem, heads):
    """Single tokens of a batch with portions go with the portions' first launch; here more sequences than travel with its arguments, and fewer."""
    for many in (130, 60):
        order = np.random.Generator(np.random.PCG64(many)).permutation(many + 5)
        check(hip, elem, [(int(s), i % 4, 1 if i % 5 else 20 + 3 * i) for i, s in enumerate(order[:many])], *heads, slots=many + 5)


@BOTH
def test_more_sequences_than_a_grid_takes(hip, elem):
    check(hip, elem, [(70000 - i, i % 3, 1) for i in range(70000)], 1, 1, 4, 4)


@BOTH
def test_samples_and_beams_of_one_prompt(hip, elem):
    """As a program uses the two together: a prompt, its state to the samples' slots, then steps before each of which every sample goes on from
    the state of a chosen one."""
    Q, H, dim, vdim, slots, n, steps = 2, 4, 64, 48, 7, 5, 12
    scale, size = np.float32(0.125), 4 * H * dim * vdim
    r = np.random.Generator(np.random.PCG64(21))
    *data, state = O.inputs(22, 90, Q, H, dim, vdim, elem, slots)
    got, st = call(hip, (*data, state), [(6, 0, 90)], elem, scale, 1e-6)
    want, exact = O.forward(*data, state, [(6, 0, 90)], scale, 1e-6)
    most = O.limit(90 + steps, dim)
    assert O.off(got, want, elem) <= most
    to, frm, at = [3, 0, 5, 1, 2], [6] * n, 90
    for step in range(steps):
        p = hip.to_device(st)
        assert hip.nvllm_copy_states(p, size, 1, slots, capi.ints(frm), capi.ints(to), n) == 0
        st = hip.to_host(p, st.shape, np.float32)
        hip.free(p)
        exact[to] = exact[frm]
        *data, _ = O.inputs(100 + step, n, Q, H, dim, vdim, elem, 1)
        spans = [(s, at, 1) for s in to]
        got, st = call(hip, (*data, st), spans, elem, scale, 1e-6)
        want, exact = O.forward(*data, exact, spans, scale, 1e-6)
        worst = O.off(got, want, elem), O.off(st[to], exact[to])
        assert max(worst) <= most, (step, worst)
        frm, at = [to[i] for i in r.integers(0, n, n)], at + 1


def test_a_captured_stream_is_refused(hip):
    """The host arrays are read at the call, so a replay would not see them; nothing is enqueued."""
    rtl = C.CDLL("libamdhip64.so")
    data = O.inputs(1, 2, 1, 1, 32, 32, O.F32, 2)
    b = Buffers(hip)
    p = [b.put(x) for x in data]
    out = b.put(np.zeros((2, 1, 32), np.float32))
    i = capi.ints([0, 1])
    hip.device_sync()
    stream, graph = C.c_void_p(hip.nvllm_stream()), C.c_void_p()
    assert rtl.hipStreamBeginCapture(stream, 0) == 0
    rc = hip.nvllm_gated_delta(out, *p, i, i, 2, 1.0, 0.0, 1, 1, 32, 32, 32, 32, 32, 4, 2)
    rs = hip.nvllm_copy_states(p[5], 4096, 1, 2, capi.ints([0]), capi.ints([1]), 1)
    assert rtl.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert (rc, rs) == (-6, -6)
    if graph.value:
        rtl.hipGraphDestroy(graph)
    hip.device_sync()
    np.testing.assert_array_equal(b.get(p[5], data[5].shape, np.float32), data[5])
    b.free()
