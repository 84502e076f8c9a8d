"""The paged 4-bit KV cache's tables and refusals, on caches without a context (no GPU)."""
import random

import pytest
from kv4_tools import Book


@pytest.fixture(scope="module")
def A():
    import aesir_hip

    return aesir_hip


def cache(A, pages=12, page=32, seqs=6, longest=300, **kw):
    a = dict(num_layers=2, n_heads=4, n_kv_heads=2, head_dim=32)
    a.update(kw)
    return A.KV4Cache(None, a["num_layers"], a["n_heads"], a["n_kv_heads"], a["head_dim"], longest, seqs, page, pages)


def same(kv, book, seqs):
    assert [kv.length(i) for i in range(seqs)] == [book.length(i) for i in range(seqs)]
    assert [kv.pages(i) for i in range(seqs)] == [book.pages(i) for i in range(seqs)]
    assert kv.free_pages == len(book.free())


@pytest.mark.parametrize("seed", range(6))
def test_random_histories_match_the_model(A, seed):
    rng = random.Random(seed)
    seqs, page = 6, 32
    pages = rng.choice([5, 12, 40])
    kv, book = cache(A, pages, page, seqs), Book(pages, page)
    refused = 0
    for _ in range(400):
        op = rng.choice(["begin"] * 4 + ["fork", "fork", "copy", "truncate", "truncate", "compact"])
        i, j = rng.randrange(seqs), rng.randrange(seqs)
        if op == "begin":
            ids = rng.sample(range(seqs), rng.randint(0, seqs))
            rows = [min(rng.choice([0, 1, 1, 3, 31, 32, 33, 70]), 300 - book.length(x)) for x in ids]
            if book.begin(ids, rows) is False:
                refused += 1
                with pytest.raises(A.AesirError) as e:
                    kv.begin(ids, rows)
                assert e.value.code == -3
            else:
                kv.begin(ids, rows)
        elif op in ("fork", "copy"):
            if book.length(j):
                with pytest.raises(A.AesirError, match="not empty"):
                    getattr(kv, op)(i, j)
            elif op == "copy" and len(book.pages(i)) > len(book.free()):
                with pytest.raises(A.AesirError) as e:
                    kv.copy(i, j)
                assert e.value.code == -3
            elif i != j:
                getattr(book, op)(i, j)
                getattr(kv, op)(i, j)
        elif op == "truncate":
            n = rng.randint(0, book.length(i))
            book.truncate(i, n)
            kv.truncate(i, n)
        else:
            assert kv.compact() == book.compact()
        same(kv, book, seqs)
    assert refused or pages == 40


def test_a_shared_last_page_is_copied_once_per_writer_but_the_last(A):
    kv = cache(A, pages=4)
    kv.begin([0], [33])
    kv.fork(0, 1)
    kv.fork(0, 2)
    assert kv.free_pages == 2
    kv.begin([0, 1, 2], [1, 0, 1])
    # sequence 1 wrote nothing and still holds page 1: both writers took a copy
    assert [kv.pages(i) for i in range(3)] == [[0, 2], [0, 1], [0, 3]]
    kv.begin([1], [1])  # now its only holder
    assert kv.pages(1) == [0, 1] and kv.free_pages == 0
    kv.truncate(0, 32)
    kv.truncate(2, 32)
    kv.fork(1, 3)
    kv.begin([1, 3], [1, 1])  # two writers, no other holder: one copy
    assert kv.pages(1) == [0, 2] and kv.pages(3) == [0, 1]


def test_a_full_last_page_is_not_copied(A):
    kv = cache(A, pages=4)
    kv.begin([0], [64])
    kv.fork(0, 1)
    kv.begin([0, 1], [1, 1])
    assert kv.pages(0) == [0, 1, 2] and kv.pages(1) == [0, 1, 3]


def test_refusals_leave_everything_as_it_was(A):
    kv = cache(A, pages=3)
    kv.begin([0], [40])
    kv.fork(0, 1)
    before = [kv.pages(i) for i in range(6)]
    for ids, rows, text in [([0, 1], [1, 40], "pages needed"), ([0, 0], [1, 1], "listed twice"), ([6], [1], "not in"), ([-1], [1], "not in"),
                            ([0], [-1], "negative"), ([0], [261], "would pass"), ([0], [1 << 62], "would pass")]:
        with pytest.raises(A.AesirError, match=text):
            kv.begin(ids, rows)
    for call, text in [(lambda: kv.fork(0, 6), "not in"), (lambda: kv.fork(-1, 2), "not in"), (lambda: kv.fork(2, 0), "not empty"),
                       (lambda: kv.copy(0, 2), "pages needed"), (lambda: kv.truncate(0, 41), "length"), (lambda: kv.truncate(0, -1), "length"),
                       (lambda: kv.truncate(9, 0), "not in"), (lambda: kv.pages(6), "out of bounds")]:
        with pytest.raises(A.AesirError, match=text):
            call()
    assert [kv.pages(i) for i in range(6)] == before and kv.free_pages == 1
    assert kv.length(6) == -1 and kv.length(-1) == -1
    kv.fork(2, 2)  # an empty sequence onto itself, and an empty one onto another: nothing to do
    kv.copy(3, 4)
    kv.begin([], [])
    assert kv.free_pages == 1


def test_sizes_are_checked(A):
    for kw, text in [(dict(num_layers=0), "positive"), (dict(n_heads=0), "positive"), (dict(page=0), "positive"), (dict(pages=-1), "positive"),
                     (dict(seqs=0), "positive"), (dict(longest=0), "positive"), (dict(n_heads=3), "multiple"), (dict(head_dim=96), "head_dim"),
                     (dict(head_dim=16), "head_dim"), (dict(page=48), "power of two"), (dict(page=16), "power of two"), (dict(page=2048), "power of two"),
                     (dict(seqs=4097), "sequences"), (dict(longest=1 << 40), "too large"), (dict(pages=1 << 40), "too large"),
                     (dict(num_layers=1 << 20), "too large"), (dict(longest=1 << 30, seqs=4096), "too large")]:
        with pytest.raises(A.AesirError, match=text):
            cache(A, **kw)
    kv = cache(A, page=64, num_layers=3, n_heads=8, n_kv_heads=4, head_dim=128)
    assert kv.page_bytes == 3 * 4 * 64 * 160  # K and V, 5 bits an element
    assert A.KV4Cache.well_bytes(3, 8, 4, 128, 300, 6, 64, 12) > 12 * kv.page_bytes
    with pytest.raises(A.AesirError, match="head_dim"):
        A.KV4Cache.well_bytes(3, 8, 4, 100, 300, 6, 64, 12)


def test_sequences_times_heads_have_a_limit(A):
    with pytest.raises(A.AesirError, match="too large"):
        cache(A, seqs=4096, n_heads=1025, n_kv_heads=1025)
    assert cache(A, seqs=4096, n_heads=1024, n_kv_heads=1024).free_pages > 0


def test_without_a_context_there_is_no_data(A):
    kv = cache(A)
    kv.begin([0], [1])
    t = A.Tensor(None, 4096, 1, 128)
    for call in (lambda: kv.append(0, t, t), lambda: kv.attention(0, t, t), lambda: kv.read(0, 1, [0], [0], [1], t, t)):
        with pytest.raises(A.AesirError, match="no context"):
            call()


def test_a_closed_context_is_not_no_context(A):
    class Closed:
        h = None

    with pytest.raises(A.AesirError, match="closed"):
        A.KV4Cache(Closed(), 1, 2, 1, 64, 64, 3, 32, 4)


def test_null_handles_are_refused(A):
    L = A._L
    assert L.aesir_kv4_begin(None, None, None, 0) == -1
    assert L.aesir_kv4_append(None, 0, None, 0, 0, None, 0, 0) == -1
    assert L.aesir_kv4_attention(None, 0, None, 0, 0, None, 0, 0) == -1
    assert L.aesir_kv4_read(None, 0, 0, None, None, None, 0, None, 0, 0, None, 0, 0) == -1
    assert L.aesir_kv4_fork(None, 0, 1) == -1 and L.aesir_kv4_copy(None, 0, 1) == -1
    assert L.aesir_kv4_truncate(None, 0, 0) == -1 and L.aesir_kv4_compact(None, None) == -1
    assert L.aesir_kv4_create(None, 1, 1, 1, 32, 32, 1, 32, 1, None) == -1
    assert L.aesir_kv4_destroy(None) == 0 and L.aesir_kv4_page_bytes(None) == -1 and L.aesir_kv4_free_pages(None) == -1
    kv = cache(A)
    assert L.aesir_kv4_begin(kv.h, None, None, 1) == -1
    assert L.aesir_kv4_pages(kv.h, 0, None, 4, None) == -1


def test_a_closed_cache_answers_no_queries(A):
    kv = cache(A)
    kv.begin([0], [5])
    kv.close()
    for call in (lambda: kv.page_bytes, lambda: kv.free_pages, lambda: kv.length(0), lambda: kv.pages(0), kv.plan, kv.compact,
                 lambda: kv.begin([0], [1]), lambda: kv.truncate(0, 0)):
        with pytest.raises(A.AesirError, match="null|closed"):
            call()
    kv.close()
