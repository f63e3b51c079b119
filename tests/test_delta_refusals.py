"""What nvllm_gated_delta refuses, before it touches the GPU: no address here is one."""
import pytest

from nvllm_amd import capi

BAD_ARGUMENT, BAD_SIZE, BAD_INDEX = -1, -2, -3


@pytest.fixture(scope="module")
def lib():
    return capi.load_hip()


GOOD = dict(out=0x1000, q=0x2000, k=0x3000, v=0x4000, g=0x5000, beta=0x6000, state=0x7000, ids=[0, 0, 1], pos=[4, 5, 0], n_slots=2, scale=1.0, eps=0.0, qk_heads=2, heads=4,
            dim=64, vdim=32, q_ld=128, k_ld=128, v_ld=128, elem=4, tokens=3)


def call(lib, **over):
    a = dict(GOOD, **over)
    ids, pos = (None if a[n] is None else capi.ints(a[n]) for n in ("ids", "pos"))
    return lib.nvllm_gated_delta(a["out"], a["q"], a["k"], a["v"], a["g"], a["beta"], a["state"], ids, pos, a["n_slots"], a["scale"], a["eps"], a["qk_heads"], a["heads"], a["dim"],
                                 a["vdim"], a["q_ld"], a["k_ld"], a["v_ld"], a["elem"], a["tokens"])


@pytest.mark.parametrize("over", [
    *[{n: None} for n in ("out", "q", "k", "v", "g", "beta", "state", "ids", "pos")],
    *[{n: bad} for n in ("n_slots", "qk_heads", "heads", "dim", "vdim") for bad in (0, -1)],
    dict(tokens=-1), dict(eps=-1e-6), dict(eps=float("nan")), dict(q_ld=127), dict(k_ld=0), dict(v_ld=127), dict(q=0x2001), dict(out=0x1002), dict(g=0x5002), dict(state=0x7001),
    dict(elem=2, k=0x3001)], ids=str)
def test_arguments(lib, over):
    assert call(lib, **over) == BAD_ARGUMENT


@pytest.mark.parametrize("over", [dict(elem=1), dict(elem=8), dict(dim=257, q_ld=514, k_ld=514), dict(heads=3, v_ld=96), dict(heads=1)], ids=str)
def test_sizes(lib, over):
    assert call(lib, **over) == BAD_SIZE


@pytest.mark.parametrize("over", [
    dict(ids=[0, 0, 2]), dict(ids=[0, 0, -1]), dict(pos=[4, 5, -1]),
    dict(pos=[4, 6, 0]), dict(pos=[4, 4, 0]), dict(pos=[5, 4, 0]),               # not one after the other
    dict(ids=[0, 1, 0], pos=[4, 0, 5]), dict(ids=[1, 1, 1], pos=[0, 1, 0])], ids=str)   # apart, twice
def test_batches(lib, over):
    assert call(lib, **over) == BAD_INDEX


@pytest.mark.parametrize("over", [dict(q_ld=2 ** 23 + 1), dict(v_ld=2 ** 23 + 8), dict(heads=2 ** 12, qk_heads=2 ** 12, dim=1, q_ld=2 ** 12, k_ld=2 ** 12, vdim=2 ** 12, v_ld=2 ** 23),
                                  dict(vdim=65536, heads=2, v_ld=2 ** 17)], ids=str)
def test_limits(lib, over):
    assert call(lib, **over) == BAD_SIZE


def test_more_sequences_than_a_call_takes(lib):
    n = 220000
    assert call(lib, ids=range(n), pos=[3] * n, n_slots=n, tokens=n) == BAD_SIZE


def test_no_tokens_is_no_call(lib):
    assert call(lib, tokens=0, out=None, ids=None) == 0
