"""Which column widths attention of a batch takes and into how many pieces it is cut, on caches without a context (no
GPU)."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def A():
    import aesir_hip

    return aesir_hip


def planned(A, hd, nq, nkv, lens, new, captured=False):
    kv = A.KV4Cache(None, 1, nq, nkv, hd, max(lens), len(lens), 64, sum(-(-x // 64) for x in lens))
    ids = list(range(len(lens)))
    kv.begin(ids, [x - r for x, r in zip(lens, new)])
    kv.begin(ids, new)
    return kv.plan(captured)


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_the_narrowest_width_that_holds_a_sequence(A, hd):
    """With much work: up to 16, 32 and 64 columns, then prompts' tiles; with little, 16-column tiles for all."""
    lens, new = [900, 300, 333, 700, 64, 40, 500], [400, 1, 16, 32, 8, 3, 5]
    assert set(planned(A, hd, 96, 48, lens, new)) == {16, 32, 64, 256}
    assert set(planned(A, hd, 96, 48, lens[1:], new[1:])) == {16, 32, 64}
    assert set(planned(A, hd, 4, 2, lens[1:], new[1:])) == {16}
    assert set(planned(A, hd, 32, 8, [2048], [130])) == {32}  # many columns, but not much work
    assert planned(A, hd, 64, 8, [7200], [61])[256] > 1 and planned(A, hd, 64, 64, [700], [700])[256] == 1


def test_head_dim_256_has_two_widths(A):
    lens, new = [900, 300, 333, 700, 64, 40, 500], [400, 1, 16, 32, 8, 3, 5]
    assert set(planned(A, 256, 96, 48, lens, new)) == {16, 128}
    assert set(planned(A, 256, 4, 2, lens[1:], new[1:])) == {16}


@pytest.mark.parametrize("hd", [64, 256])
def test_a_captured_call_is_one_launch_as_wide_as_the_widest(A, hd):
    lens, new = [900, 300, 333, 700, 64, 40, 500], [400, 1, 16, 32, 8, 3, 5]
    for n in (0, 1, 4, 5, 6):
        eager = planned(A, hd, 96, 48, lens[n:], new[n:])
        assert list(planned(A, hd, 96, 48, lens[n:], new[n:], captured=True)) == [max(eager)]


def test_no_batch_and_no_rows_have_no_launch(A):
    kv = A.KV4Cache(None, 1, 4, 2, 64, 300, 3, 32, 12)
    assert kv.plan() == {} and kv.plan(captured=True) == {}
    kv.begin([0, 1], [0, 0])
    assert kv.plan() == {}
    kv.begin([0, 1], [0, 1])
    assert kv.plan() == {16: 1}
    kv.truncate(2, 0)
    assert kv.plan() == {}


def test_bad_arguments(A):
    L, n = A._L, C.c_int64()
    kv = A.KV4Cache(None, 1, 4, 2, 64, 300, 3, 32, 12)
    kv.begin([0], [1])
    assert L.aesir_kv4_plan(None, 0, None, None, 0, C.byref(n)) == -1 and L.aesir_kv4_plan(kv.h, 0, None, None, 0, None) == -1
    assert L.aesir_kv4_plan(kv.h, 0, None, None, 1, C.byref(n)) == -1 and L.aesir_kv4_plan(kv.h, 0, None, None, -1, C.byref(n)) == -1
    assert L.aesir_kv4_plan(kv.h, 0, None, None, 0, C.byref(n)) == 0 and n.value == 1
