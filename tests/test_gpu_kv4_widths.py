"""Attention of the paged 4-bit KV cache in every column width and head_dim, each test stating the widths that it is
about (KV4Cache.plan): tiles whole and cut, column remainders, inf and NaN in and behind rows, mixed batches, and captured
launches of each width that serve other batches."""
import numpy as np
import pytest
from kv4_tools import kv4_values
from test_gpu_kv4 import A, Graph, _well, attend, ctx  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu

WIDE = {32: 256, 64: 256, 128: 256, 256: 128}  # columns of a prompt's tile


def rand(rng, *shape):
    return rng.standard_normal(shape, dtype=np.float32).astype(np.float16)


def cache(A, ctx, hd, nq, nkv, lens, page=64):
    return A.KV4Cache(ctx, 1, nq, nkv, hd, max(lens), len(lens), page, sum(-(-x // page) for x in lens))


def fill(ctx, kv, ids, data, lens, new):
    """Every sequence's earlier positions, then the batch of its new ones."""
    for rows in ([x - r for x, r in zip(lens, new)], new):
        kv.begin(ids, rows)
        mark = ctx.offset
        if sum(rows):
            first = rows is not new
            part = [[x[:n - r] if first else x[n - r:n] for x in d] for d, n, r in zip(data, lens, new)]
            kv.append(0, *(ctx.from_numpy(np.concatenate([p[j] for p in part])) for j in (0, 1)))
        ctx.synchronize()
        ctx.reset(mark)


def expect(q, K, V):
    """Output of query rows q [G, hd] over value rows K and V in 64 bits, and how far an f16 output may be off: half an f16
    step; every weight's rounding to f16 (2^-11) and the f32 roundings of its score, exponential and the sums, doubled, each
    against the distance of its value from the output; and weights under 2^-39 of the largest."""
    hd, S = q.shape[1], len(K)
    q, K, V = (x.astype(np.float64) for x in (q, K, V))
    s = q @ K.T / np.sqrt(hd)
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    want = p @ V
    top = (np.abs(q) @ np.abs(K).T).max(1, keepdims=True) / np.sqrt(hd)
    spread = p @ np.abs(V) + np.abs(want)
    half = np.spacing(np.abs(want).astype(np.float16)).astype(np.float64) / 2
    return want, half * (1 + 2.0 ** -9) + spread * (2.0 ** -11 + ((hd + 16) * (1 + top) + S) * 2.0 ** -23) + S * 2.0 ** -39 * np.abs(V).max()


def some(n):
    return sorted({0, 1, n // 2, n - 2, n - 1} & set(range(n)))


def check(got, q, data, lens, new, hd, nq, nkv, served=None):
    """A few rows and KV heads of every sequence; served: only the first rows of the batch."""
    G, at = nq // nkv, 0
    for (k, v), n, r in zip(data, lens, new):
        for h in sorted({0, nkv // 2, nkv - 1}):
            c = slice(h * hd, (h + 1) * hd)
            K, V = kv4_values(k[:n, c]), kv4_values(v[:n, c])
            for j in some(r):
                if served is not None and at + j >= served:
                    continue
                w = slice(h * G * hd, (h + 1) * G * hd)
                x = q[at + j, w].reshape(G, hd)
                want, bound = expect(x, K[:n - r + j + 1], V[:n - r + j + 1])
                off = np.abs(got[at + j, w].reshape(G, hd) - want) - bound
                assert (off <= 0).all(), (at, j, h, float(off.max()), float(bound.max()))
        at += r


WHOLE, CUT = (64, 64, 700, 700), (64, 8, 7200, 61)  # nq, nkv, positions, rows


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("nq,nkv,length,rows", [WHOLE, CUT, (60, 12, 3001, 333)])
def test_prompts(A, ctx, hd, nq, nkv, length, rows):
    """Prompts' tiles whole and cut, the last one in part."""
    rng = np.random.default_rng(hd)
    kv = cache(A, ctx, hd, nq, nkv, [length])
    data = [(rand(rng, length, nkv * hd), rand(rng, length, nkv * hd))]
    fill(ctx, kv, [0], data, [length], [rows])
    plan = kv.plan()
    assert list(plan) == [WIDE[hd]] and rows * nq // nkv % WIDE[hd]
    if (nq, nkv, length, rows) == WHOLE:
        assert plan[WIDE[hd]] == 1
    if (nq, nkv, length, rows) == CUT:
        assert plan[WIDE[hd]] > 1
    q = rand(rng, rows, nq * hd)
    got = attend(A, ctx, kv, 0, q)
    check(got, q, data, [length], [rows], hd, nq, nkv)
    assert np.array_equal(got, attend(A, ctx, kv, 0, q))


SHAPES = [(16, (64, 8, 900, 2)), (32, (32, 8, 8192, 8)), (64, (32, 8, 8192, 16)), (0, WHOLE), (0, CUT)]


def there_is(hd, width):
    return hd < 256 or width not in (32, 64)


@pytest.mark.parametrize("hd,width,shape", [(hd, w, s) for hd in WIDE for w, s in SHAPES if there_is(hd, w)])
def test_inf_and_nan_reach_the_rows_that_see_them(A, ctx, hd, width, shape):
    """Freed pages full of NaN under the sequence's, and new rows with inf and NaN: outputs are NaN where a row's own
    positions say so and those of the other positions elsewhere."""
    nq, nkv, length, rows = shape
    rng, G = np.random.default_rng(hd + rows), nq // nkv
    kv = cache(A, ctx, hd, nq, nkv, [length + 64])
    bad = np.full((1, nkv * hd), np.nan, np.float16)
    kv.begin([0], [length + 64])
    mark = ctx.offset
    nan = ctx.from_numpy(np.repeat(bad, length + 64, 0))
    kv.append(0, nan, nan)
    ctx.synchronize()
    ctx.reset(mark)
    kv.truncate(0, 0)
    k, v = rand(rng, length, nkv * hd), rand(rng, length, nkv * hd)
    # positions of the batch's rows: a NaN key of head 0, an inf in head 1's first 32 values, a NaN in its last 32 and one in
    # the last head's, in rows of their own where there are enough
    at = [rows // 4, rows // 2, rows // 2 + rows // 8, rows - 1]
    p = [length - rows + x for x in at]
    k[p[0], 3] = np.nan
    v[p[1], hd + 2] = np.inf
    v[p[2], 2 * hd - 1] = np.nan
    v[p[3], -1] = -np.inf
    fill(ctx, kv, [0], [(k, v)], [length], [rows])
    assert list(kv.plan()) == [width or WIDE[hd]]
    q = rand(rng, rows, nq * hd)
    got = attend(A, ctx, kv, 0, q).reshape(rows, nkv, G, hd)
    want = np.zeros(got.shape, bool)
    want[at[0]:, 0] = True
    want[at[1]:, 1, :, :32] = True
    want[at[2]:, 1, :, -32:] = True
    want[at[3]:, -1, :, -32:] = True
    assert np.array_equal(np.isnan(got), want), np.argwhere(np.isnan(got) != want)[:5]
    q = q.reshape(rows, nkv, G, hd)
    for h in sorted({0, 1, 2, nkv - 1}):
        c = slice(h * hd, (h + 1) * hd)
        K, V = kv4_values(k[:, c]), kv4_values(v[:, c])
        for j in sorted(set(some(rows) + [x - 1 for x in at if x > 0])):
            n = length - rows + j + 1
            if h == 0 and j >= at[0]:
                continue
            x, bound = expect(q[j, h], K[:n], np.nan_to_num(V[:n]))
            ok = ~want[j, h]
            assert (np.abs(got[j, h] - x)[ok] <= bound[ok]).all(), (h, j)


MIXED = ([900, 300, 333, 700, 64, 40, 500], [400, 1, 16, 32, 8, 3, 5])


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("first", [0, 1, 3])
def test_batches_of_all_widths(A, ctx, hd, first):
    """Every width in one batch; without prompts; without 32 columns; eagerly and captured."""
    rng = np.random.default_rng(hd + first)
    nq, nkv = 96, 48
    lens, new = (x[first:] for x in MIXED)
    kv = cache(A, ctx, hd, nq, nkv, lens)
    data = [(rand(rng, n, nkv * hd), rand(rng, n, nkv * hd)) for n in lens]
    ids = list(range(len(lens)))
    fill(ctx, kv, ids, data, lens, new)
    want = {0: {16, 32, 64, 256}, 1: {16, 32, 64}, 3: {16, 64}} if hd < 256 else {0: {16, 128}, 1: {16, 128}, 3: {16}}
    want = want[first]
    assert set(kv.plan()) == want and list(kv.plan(captured=True)) == [max(want)]
    q = rand(rng, sum(new), nq * hd)
    check(attend(A, ctx, kv, 0, q), q, data, lens, new, hd, nq, nkv)
    tq, out = ctx.from_numpy(q), ctx.from_numpy(np.zeros_like(q))
    g = Graph(A, ctx, lambda: kv.attention(0, tq, out))
    for _ in range(3):
        out.upload(np.zeros_like(q))
        g.launch()
        check(out.numpy().astype(np.float64), q, data, lens, new, hd, nq, nkv)
    g.close()


@pytest.mark.parametrize("hd,width,rows", [(hd, w, r) for hd in WIDE for w, r in [(16, 1), (32, 8), (64, 16), (0, 128)] if there_is(hd, w)])
def test_a_captured_launch_of_each_width_serves_other_batches(A, ctx, hd, width, rows):
    """Captured for one long sequence; replayed for batches of fewer and of more rows than the capture had, shorter and
    longer, for none, and again for its own, with eager calls between."""
    rng = np.random.default_rng(hd + rows)
    nq, nkv, seqs = 32, 8, 5
    kv = A.KV4Cache(ctx, 1, nq, nkv, hd, 8192, seqs, 64, 200)
    data = [(rand(rng, 8192, nkv * hd), rand(rng, 8192, nkv * hd))] + [(rand(rng, 3000, nkv * hd), rand(rng, 3000, nkv * hd)) for _ in range(4)]
    q, out = ctx.tensor(rows, nq * hd), ctx.tensor(rows, nq * hd)
    fill(ctx, kv, [0], data[:1], [8192], [rows])
    width = width or WIDE[hd]
    assert list(kv.plan(captured=True)) == [width]
    g = Graph(A, ctx, lambda: kv.attention(0, q, out))
    one = ([0], [8192], [rows])
    steps = [one, ([3, 1], [700, 33], [0, 1]), ([2], [2999], [rows]), ([4, 2, 1, 3], [1000, 64, 2500, 300], [-(-rows // 4)] * 4),
             ([1, 2], [3000, 1500], [max(1, rows // 2), 2 * rows]), ([3], [64 + 3 * rows], [3 * rows]), one]
    for ids, lens, new in steps:
        for i in range(seqs):
            kv.truncate(i, 0)
        out.upload(np.full((rows, nq * hd), 9.0, np.float16))
        g.launch()  # no batch: nothing is written
        assert (out.numpy() == 9.0).all()
        mine, n = [data[i] for i in ids], sum(new)
        fill(ctx, kv, ids, mine, lens, new)
        x = rand(rng, max(n, rows), nq * hd)
        q.upload(x[:rows])
        for _ in range(2):
            out.upload(np.full((rows, nq * hd), 9.0, np.float16))
            g.launch()
            got = out.numpy().astype(np.float64)
            check(got, x, mine, lens, new, hd, nq, nkv, served=rows)
            assert (got[n:] == 9.0).all()
            mark = ctx.offset
            check(attend(A, ctx, kv, 0, x[:n]), x, mine, lens, new, hd, nq, nkv)
            ctx.reset(mark)
    g.close()
