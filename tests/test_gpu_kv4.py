"""The paged 4-bit KV cache on the GPU: stored values bit for bit, attention against 64 bits within derived
bounds, page operations, captured calls, and what a batch must leave alone."""
import ctypes as C
import random

import numpy as np
import pytest
from kv4_tools import attention64, attention_bound, kv4_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A():
    import aesir_hip

    return aesir_hip


@pytest.fixture(scope="module")
def ctx(A):
    with A.Context(2 << 30) as c:
        yield c


@pytest.fixture(autouse=True)
def _well(ctx):
    mark = ctx.offset
    yield
    ctx.reset(mark)


def rand(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


def attend(A, ctx, kv, layer, q):
    out = ctx.from_numpy(np.full_like(q, 7.0))
    kv.attention(layer, ctx.from_numpy(q), out)
    return out.numpy().astype(np.float64)


def read(ctx, kv, layer, layers, seqs, pos, rows):
    n, w = layers * sum(rows), kv.n_kv_heads * kv.head_dim
    k, v = ctx.tensor(n, w), ctx.tensor(n, w)
    kv.read(layer, layers, seqs, pos, rows, k, v)
    return k.numpy(), v.numpy()


def same_bits(got, want):
    """Equal values (a zero's sign aside), NaN where NaN."""
    g, w = got.astype(np.float64), want.astype(np.float64)
    ok = (g == w) | (np.isnan(g) & np.isnan(w))
    assert ok.all(), (np.argwhere(~ok)[:3], got[~ok][:3], want[~ok][:3])


def check(got, q, K, V, nq, nkv, hd):
    """got [rows, nq hd] against attention over value rows K and V."""
    want, mass, top = attention64(q, K, V, nq, nkv, hd)
    bound = attention_bound(want, mass, top, len(K), hd, np.abs(V.astype(np.float64)).max())
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), (np.unravel_index(off.argmax(), off.shape), float(off.max()), float(bound.max()))


# ------------------------------------------------------------------ stored values

@pytest.mark.parametrize("hd,nkv,page", [(32, 1, 32), (32, 5, 64), (64, 3, 32), (64, 4, 128), (128, 8, 64), (128, 1, 1024), (256, 2, 32), (256, 3, 64)])
def test_values_come_back_as_defined(A, ctx, hd, nkv, page):
    """Ragged batches at uneven positions, rows of many kinds; every layer keeps its own."""
    rng = np.random.default_rng(hd + nkv)
    kv = A.KV4Cache(ctx, 2, nkv, nkv, hd, 500, 5, page, 5 * -(-500 // page))
    have = {i: [[np.empty((0, nkv * hd), np.float16)] * 2 for _ in range(2)] for i in range(5)}
    for ids, rows in [([3], [1]), ([0, 3, 1], [45, 2, 0]), ([1, 0, 4, 3], [3, 1, 130, 64]), ([4, 2], [1, 7])]:
        kv.begin(ids, rows)
        for layer in range(2):
            k, v = rand(rng, sum(rows), nkv * hd), rand(rng, sum(rows), nkv * hd)
            k *= np.exp(2 * rng.standard_normal((1, nkv * hd))).astype(np.float16)
            kv.append(layer, ctx.from_numpy(k), ctx.from_numpy(v))
            at = 0
            for i, r in zip(ids, rows):
                have[i][layer] = [np.concatenate([x, y[at:at + r]]) for x, y in zip(have[i][layer], (k, v))]
                at += r
    lens = [kv.length(i) for i in range(5)]
    assert lens == [len(have[i][0][0]) for i in range(5)]
    got = read(ctx, kv, 0, 2, [4, 0, 1, 2, 3], [0] * 5, [lens[i] for i in (4, 0, 1, 2, 3)])
    for j in range(2):
        want = np.concatenate([have[i][layer][j] for layer in range(2) for i in (4, 0, 1, 2, 3)])
        same_bits(got[j], kv4_values(want))
    got = read(ctx, kv, 1, 1, [0, 0, 4], [lens[0], 31, 33], [0, 15, 97])  # ranges, a sequence twice, an empty one
    for j in range(2):
        same_bits(got[j], kv4_values(np.concatenate([have[0][1][j][31:46], have[4][1][j][33:130]])))


def special_rows(rng, hd):
    """Rows whose groups meet the rounding rules' corners."""
    def group(*x):
        return np.resize(np.array(x, np.float16), 32)
    tiny = np.float16(2.0 ** -24)
    g = [group(0.0), group(-0.0, 0.0), group(3.25), group(65504, -65504), group(65504, 65472, -65504), group(-65504, 65504, 1.0, 0.5),
         group(*(tiny * np.arange(32).astype(np.float16))), group(0, tiny), group(0, tiny * 7), group(0, tiny * 8), group(1, np.float16(1.001)),
         group(*np.arange(0, 16)), group(*(np.arange(0, 31) / 2)), group(-7.5, 7.5, 0.0, tiny, -tiny, 1e-5), group(960, tiny, 0.0), group(-1000, 1e-6, 1000, 0),
         group(np.inf, 1), group(-np.inf), group(np.nan, 2), group(1875 / 1000, -1875 / 1000, 0, tiny, -tiny), group(*np.linspace(-1, 1, 32))]
    g += [np.float16(s) * rand(rng, 32) for s in (1e-6, 1e-4, 1e-2, 1, 100, 1e4)]
    # quotients on and beside the borders between levels
    for d in (0.125, 0.3, 7.0):
        d = np.float16(d)
        mid = (np.arange(15) + 0.5) * float(d)
        mids = mid.astype(np.float16)
        g += [group(0, d * np.float16(15), *mids), group(0, d * np.float16(15), *np.nextafter(mids, np.float16(9e4))),
              group(0, d * np.float16(15), *np.nextafter(mids, np.float16(-9e4)))]
    while len(g) % (hd // 32):
        g.append(group(1, 2))
    return np.stack(g).reshape(-1, hd)


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_corner_values(A, ctx, hd):
    rng = np.random.default_rng(1)
    k = special_rows(rng, hd)
    v = np.ascontiguousarray(k[::-1])
    kv = A.KV4Cache(ctx, 1, 1, 1, hd, len(k), 1, 32, -(-len(k) // 32))
    kv.begin([0], [len(k)])
    kv.append(0, ctx.from_numpy(k), ctx.from_numpy(v))
    got = read(ctx, kv, 0, 1, [0], [0], [len(k)])
    for g, x in zip(got, (k, v)):
        same_bits(g, kv4_values(x))
        fin = np.isfinite(x.reshape(-1, 32)).all(1)
        gg, xx = g.reshape(-1, 32)[fin].astype(np.float64), x.reshape(-1, 32)[fin].astype(np.float64)
        step = (xx.max(1) - xx.min(1)) / 15 * (1 + 2.0 ** -10)
        limit = np.maximum(step / 2, 15 * 2.0 ** -25)[:, None] + np.spacing(np.abs(gg).astype(np.float16)).astype(np.float64)
        assert (np.abs(gg - xx) <= limit).all()


@pytest.mark.parametrize("offset,pad", [(1, 0), (0, 3), (8, 8), (5, 11)])
def test_views_of_wider_rows(A, ctx, offset, pad):
    """K, V, Q and outputs inside wider matrices, aligned or not; the columns around them stay as they were."""
    rng = np.random.default_rng(offset + pad)
    nq, nkv, hd, rows = 4, 2, 64, 9
    w, wq = nkv * hd, nq * hd
    kv = A.KV4Cache(ctx, 1, nq, nkv, hd, 64, 1, 32, 2)

    def wide(x):
        n = x.shape[1] + pad
        m = np.full(rows * n + offset, 3.0, np.float16)
        m[offset:].reshape(rows, n)[:, :x.shape[1]] = x
        return ctx.from_numpy(m.reshape(1, -1)).view(rows, n, offset), m

    k, v, q = rand(rng, rows, w), rand(rng, rows, w), rand(rng, rows, wq)
    kv.begin([0], [rows])
    kv.append(0, wide(k)[0], wide(v)[0])
    o, om = wide(np.zeros((rows, wq), np.float16))
    kv.attention(0, wide(q)[0], o)
    got = o.numpy()
    check(got[:, :wq].astype(np.float64), q, kv4_values(k), kv4_values(v), nq, nkv, hd)
    assert (got[:, wq:][:-1] == 3.0).all()
    (kb, _), (vb, _) = wide(np.zeros((rows, w), np.float16)), wide(np.zeros((rows, w), np.float16))
    kv.read(0, 1, [0], [0], [rows], kb, vb)
    for t, x in ((kb, k), (vb, v)):
        same_bits(t.numpy()[:, :w], kv4_values(x))
        assert (t.numpy()[:, w:][:-1] == 3.0).all()


# ------------------------------------------------------------------ attention

SHAPES = [(32, 8, 2), (64, 32, 4), (128, 32, 8), (128, 4, 4), (128, 12, 4), (256, 8, 2), (64, 5, 1), (64, 40, 2), (32, 3, 3)]


@pytest.mark.parametrize("hd,nq,nkv", SHAPES)
@pytest.mark.parametrize("page", [32, 64])
def test_attention_of_ragged_batches(A, ctx, hd, nq, nkv, page):
    """Lengths around a page, a 32-key round and a split, from one position; 0, 1 and several new rows."""
    rng = np.random.default_rng(hd * nq + page)
    lens = [1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 300, 517, 5, 40]
    new = [1, 2, 1, 5, 1, 1, 0, 1, 3, 1, 1, 17, 5, 40]
    n = len(lens)
    kv = A.KV4Cache(ctx, 2, nq, nkv, hd, 600, n, page, sum(-(-x // page) for x in lens))
    data = [(rand(rng, x, nkv * hd), rand(rng, x, nkv * hd)) for x in lens]
    ids = list(range(n))
    kv.begin(ids, [x - r for x, r in zip(lens, new)])
    kv.append(1, *(ctx.from_numpy(np.concatenate([d[j][:x - r] for d, x, r in zip(data, lens, new)])) for j in (0, 1)))
    order = ids[::-1]
    kv.begin(order, [new[i] for i in order])
    kv.append(1, *(ctx.from_numpy(np.concatenate([data[i][j][lens[i] - new[i]:] for i in order])) for j in (0, 1)))
    q = rand(rng, sum(new), nq * hd)
    got = attend(A, ctx, kv, 1, q)
    at = 0
    for i in order:
        if new[i]:
            check(got[at:at + new[i]], q[at:at + new[i]], kv4_values(data[i][0]), kv4_values(data[i][1]), nq, nkv, hd)
        at += new[i]


@pytest.mark.parametrize("hd,nq,nkv,length,rows", [(128, 8, 2, 5000, 1), (64, 8, 1, 3001, 4), (128, 4, 4, 2100, 1), (256, 2, 1, 1500, 3), (32, 16, 1, 2000, 1),
                                                   (128, 4, 1, 700, 230), (64, 8, 1, 333, 333), (256, 2, 1, 300, 70), (32, 4, 2, 200, 101)])
def test_attention_of_long_and_wide_batches(A, ctx, hd, nq, nkv, length, rows):
    rng = np.random.default_rng(length + rows)
    kv = A.KV4Cache(ctx, 1, nq, nkv, hd, length, 1, 64, -(-length // 64))
    k, v, q = rand(rng, length, nkv * hd), rand(rng, length, nkv * hd), rand(rng, rows, nq * hd)
    q *= np.float16(2.0)
    kv.begin([0], [length - rows])
    if length > rows:
        kv.append(0, ctx.from_numpy(k[:-rows]), ctx.from_numpy(v[:-rows]))
    kv.begin([0], [rows])
    kv.append(0, ctx.from_numpy(k[-rows:]), ctx.from_numpy(v[-rows:]))
    got = attend(A, ctx, kv, 0, q)
    some = sorted(set([0, 1, rows // 2, rows - 1]) & set(range(rows)))
    for r in some:
        n = length - rows + r + 1
        check(got[r:r + 1], q[r:r + 1], kv4_values(k[:n]), kv4_values(v[:n]), nq, nkv, hd)
    again = attend(A, ctx, kv, 0, q)
    assert np.array_equal(got, again)  # the order of every sum is fixed


@pytest.mark.parametrize("hd,nq,nkv,lens,new", [
    (32, 128, 128, [3500, 1200, 3300, 700, 2600], [1, 1, 1, 1, 1]),      # equal shares that cut and join tiles of 16
    (64, 96, 96, [3200, 3100, 1900], [1, 3, 1]),                         # a workgroup to a piece
    (32, 256, 64, [3300, 3150, 700, 1800], [6, 5, 8, 7]),                # shares of 32-column tiles
    (64, 128, 16, [4000, 3300, 900, 2500, 3900, 3600, 1300], [6] * 7),   # of 64-column tiles
    (256, 16, 16, [3900, 2500, 3700, 1300, 3300, 100], [1] * 6)])
def test_attention_cut_into_equal_shares(A, ctx, hd, nq, nkv, lens, new):
    """More work than the workgroups that run at once take as pieces of their own: a few heads of every row."""
    rng = np.random.default_rng(nkv)
    ids = list(range(len(lens)))
    kv = A.KV4Cache(ctx, 1, nq, nkv, hd, 4096, len(ids), 128, sum(-(-x // 128) for x in lens))
    data = [rng.standard_normal((2, x, nkv * hd), dtype=np.float32).astype(np.float16) for x in lens]
    kv.begin(ids, [x - r for x, r in zip(lens, new)])
    mark = ctx.offset
    kv.append(0, *(ctx.from_numpy(np.concatenate([d[j, :x - r] for d, x, r in zip(data, lens, new)])) for j in (0, 1)))
    ctx.reset(mark)
    kv.begin(ids, new)
    kv.append(0, *(ctx.from_numpy(np.concatenate([d[j, x - r:] for d, x, r in zip(data, lens, new)])) for j in (0, 1)))
    q = rand(rng, sum(new), nq * hd)
    got = attend(A, ctx, kv, 0, q).reshape(sum(new), nkv, -1)
    at = 0
    for d, r in zip(data, new):
        for h in (0, nkv // 2 + 1, nkv - 1):
            K, V = (kv4_values(x[:, h * hd:(h + 1) * hd]) for x in d)
            w = nq // nkv * hd
            check(got[at:at + r, h], q[at:at + r, h * w:(h + 1) * w], K, V, nq // nkv, 1, hd)
        at += r


@pytest.mark.parametrize("where", ["first", "last", "middle"])
def test_a_probability_near_one_and_many_tiny_ones(A, ctx, where):
    """One key 16 above 4095 others (each 2^-23 of it, 2^-11 together): their sum is not lost."""
    hd, S = 64, 4096
    k, v = np.zeros((S, hd), np.float16), np.full((S, hd), 512.0, np.float16)
    v[:, ::2] = -512.0
    at = {"first": 0, "last": S - 1, "middle": 2047}[where]
    k[at, :] = 16.0  # score 16 * 64 * q / 8
    v[at] = 0
    q = np.full((1, hd), 0.125, np.float16)
    kv = A.KV4Cache(ctx, 1, 1, 1, hd, S, 1, 64, S // 64)
    kv.begin([0], [S - 1])
    kv.append(0, ctx.from_numpy(k[:-1]), ctx.from_numpy(v[:-1]))
    kv.begin([0], [1])
    kv.append(0, ctx.from_numpy(k[-1:]), ctx.from_numpy(v[-1:]))
    check(attend(A, ctx, kv, 0, q), q, kv4_values(k), kv4_values(v), 1, 1, hd)


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("nq", [2, 4, 32])
def test_nothing_behind_a_row_reaches_it(A, ctx, hd, nq):
    """Freed pages full of NaN under the next sequence's last page, and later rows of the same batch whose
    keys and values are inf or NaN: a row's output is that of its own positions."""
    rng = np.random.default_rng(hd)
    nkv, rows, S = 2, 24, 70
    kv = A.KV4Cache(ctx, 1, nq, nkv, hd, 128, 1, 64, 2)
    bad = np.full((128, nkv * hd), np.nan, np.float16)
    kv.begin([0], [128])
    kv.append(0, ctx.from_numpy(bad), ctx.from_numpy(bad))
    kv.truncate(0, 0)
    k, v, q = rand(rng, S, nkv * hd), rand(rng, S, nkv * hd), rand(rng, rows, nq * hd)
    k[S - 10, 3] = np.nan       # row 14's own key: head 0's scores of rows 14 .. are NaN
    v[S - 6, hd] = np.inf       # row 18's own value: head 1's first 32 dims
    v[S - 4, hd - 1] = np.nan   # row 20's: head 0's last 32 dims
    kv.begin([0], [S - rows])
    kv.append(0, ctx.from_numpy(k[:S - rows]), ctx.from_numpy(v[:S - rows]))
    kv.begin([0], [rows])
    kv.append(0, ctx.from_numpy(k[S - rows:]), ctx.from_numpy(v[S - rows:]))
    got = attend(A, ctx, kv, 0, q).reshape(rows, nq, hd)
    K, V = kv4_values(k), kv4_values(v)
    want_nan = np.zeros((rows, nq, hd), bool)
    want_nan[14:, :nq // 2] = True          # the query heads of KV head 0
    want_nan[18:, nq // 2:, :32] = True
    assert np.array_equal(np.isnan(got), want_nan), np.argwhere(np.isnan(got) != want_nan)[:5]
    Vc = V.copy()
    Vc[S - 6, hd:hd + 32] = 0               # for the dims that stay finite
    for r in range(rows):
        n = S - rows + r + 1
        w, mass, top = attention64(q[r:r + 1], np.nan_to_num(K[:n]), np.nan_to_num(Vc[:n]), nq, nkv, hd)
        b = attention_bound(w, mass, top, n, hd, 8.0)
        ok = ~want_nan[r].reshape(-1)
        assert (np.abs(got[r].reshape(-1) - w[0])[ok] <= b[0][ok]).all(), r


@pytest.mark.parametrize("hd,nq,nkv", [(32, 8, 2), (64, 8, 1), (128, 8, 2), (256, 4, 1), (128, 3, 3)])
def test_batches_of_prompts_drafts_and_single_rows(A, ctx, hd, nq, nkv):
    """Sequences of every column class in one batch, short and long, and a captured call of the same."""
    rng = np.random.default_rng(hd + nq)
    lens, new = [700, 300, 520, 900, 64, 2000, 33, 90], [1, 7, 40, 130, 64, 1, 2, 11]
    ids = list(range(len(lens)))
    kv = A.KV4Cache(ctx, 1, nq, nkv, hd, 2048, len(ids), 64, sum(-(-x // 64) for x in lens))
    data = [(rand(rng, x, nkv * hd), rand(rng, x, nkv * hd)) for x in lens]
    kv.begin(ids, [x - r for x, r in zip(lens, new)])
    kv.append(0, *(ctx.from_numpy(np.concatenate([d[j][:x - r] for d, x, r in zip(data, lens, new)])) for j in (0, 1)))
    kv.begin(ids, new)
    kv.append(0, *(ctx.from_numpy(np.concatenate([d[j][x - r:] for d, x, r in zip(data, lens, new)])) for j in (0, 1)))
    q = rand(rng, sum(new), nq * hd)
    got = attend(A, ctx, kv, 0, q)
    tq, out = ctx.from_numpy(q), ctx.from_numpy(np.zeros_like(q))
    g = Graph(A, ctx, lambda: kv.attention(0, tq, out))
    g.launch()
    again = out.numpy().astype(np.float64)
    g.close()
    at = 0
    for (k, v), x, r in zip(data, lens, new):
        K, V = kv4_values(k), kv4_values(v)
        for j in sorted({0, 1, r // 2, r - 1} & set(range(r))):
            for o in (got, again):
                check(o[at + j:at + j + 1], q[at + j:at + j + 1], K[:x - r + j + 1], V[:x - r + j + 1], nq, nkv, hd)
        at += r


@pytest.mark.parametrize("rows", [1, 3, 8, 80])
@pytest.mark.parametrize("size", [30.0, 3000.0, 60000.0])
def test_scores_of_any_size(A, ctx, rows, size):
    """Scores from hundreds to the largest f16 rows give (10^10): no probability overflows, and a row whose best key
    is alone gets its value. Keys are multiples of one row, so that products are exact: q = size, keys +-size times 0,
    2^-6, .., values that tell them apart."""
    nq, nkv, hd, S = 8, 2, 64, 300
    rng = np.random.default_rng(rows)
    steps = rng.permutation(np.concatenate([-np.arange(150), np.arange(150)])).astype(np.float64) / 150
    k = np.repeat((steps * size)[:, None], nkv * hd, 1).astype(np.float16)
    v = rand(rng, S, nkv * hd)
    q = np.full((rows, nq * hd), size, np.float16)
    q[:, hd:2 * hd] *= -1
    kv = A.KV4Cache(ctx, 1, nq, nkv, hd, S, 1, 32, 10)
    kv.begin([0], [S - rows])
    kv.append(0, ctx.from_numpy(k[:S - rows]), ctx.from_numpy(v[:S - rows]))
    kv.begin([0], [rows])
    kv.append(0, ctx.from_numpy(k[S - rows:]), ctx.from_numpy(v[S - rows:]))
    got = attend(A, ctx, kv, 0, q)
    K, V = kv4_values(k), kv4_values(v).astype(np.float64).reshape(S, nkv, hd)
    for r in range(rows):
        n = S - rows + r + 1
        for h in range(nq):
            z = K[:n, 0].astype(np.float64) * q[r, h * hd].astype(np.float64) * hd / 8
            if np.sort(z)[-1] - np.sort(z)[-2] > 60:  # e^-60 of the others is below every rounding
                assert np.abs(got[r, h * hd:(h + 1) * hd] - V[z.argmax(), h // 4]).max() <= 2.0 ** -10 * np.abs(V).max(), (r, h)
            assert np.isfinite(got[r, h * hd:(h + 1) * hd]).all()


def test_a_bad_query_row_is_its_own(A, ctx):
    rng = np.random.default_rng(2)
    nq, nkv, hd, rows = 4, 1, 128, 6
    kv = A.KV4Cache(ctx, 1, nq, nkv, hd, 64, 1, 32, 2)
    k, v, q = rand(rng, rows, hd), rand(rng, rows, hd), rand(rng, rows, nq * hd)
    q[2, hd + 5], q[4, 0] = np.nan, np.inf
    kv.begin([0], [rows])
    kv.append(0, ctx.from_numpy(k), ctx.from_numpy(v))
    got = attend(A, ctx, kv, 0, q).reshape(rows, nq, hd)
    nan = np.isnan(got)
    assert nan[2, 1].all() and not nan[2, [0, 2, 3]].any() and nan[4, 0].all() and not nan[4, 1:].any()
    q[2, hd + 5], q[4, 0] = 0, 0
    clean = attend(A, ctx, kv, 0, q).reshape(rows, nq, hd)
    assert np.array_equal(got[~nan], clean[~nan])


def test_equal_values_come_out_equal(A, ctx):
    """Weights of a row sum to one: rows of one value give it back, within one probability rounding."""
    hd, S = 128, 777
    rng = np.random.default_rng(3)
    kv = A.KV4Cache(ctx, 1, 8, 2, hd, S, 1, 64, 13)
    k, v = rand(rng, S, 2 * hd), np.full((S, 2 * hd), 1.5, np.float16)
    kv.begin([0], [S])
    kv.append(0, ctx.from_numpy(k), ctx.from_numpy(v))
    got = attend(A, ctx, kv, 0, rand(rng, S, 8 * hd))
    assert np.abs(got - 1.5).max() <= 1.5 * 2.0 ** -11 + 2.0 ** -10


def test_many_sequences(A, ctx):
    """300 sequences of one head in one batch, every third without a new row."""
    rng = np.random.default_rng(4)
    nq, nkv, hd, n = 2, 1, 64, 300
    lens = [1 + (37 * i) % 90 for i in range(n)]
    kv = A.KV4Cache(ctx, 1, nq, nkv, hd, 128, n, 32, 3 * n)
    k, v = rand(rng, sum(lens), hd), rand(rng, sum(lens), hd)
    start = np.concatenate([[0], np.cumsum(lens)])
    ids = list(range(n))
    new = [0 if i % 3 == 0 else 1 for i in ids]
    early = [np.concatenate([x[start[i]:start[i + 1] - new[i]] for i in ids]) for x in (k, v)]
    kv.begin(ids, [a - b for a, b in zip(lens, new)])
    kv.append(0, *map(ctx.from_numpy, early))
    kv.begin(ids, new)
    last = [np.concatenate([x[start[i + 1] - new[i]:start[i + 1]] for i in ids]) for x in (k, v)]
    kv.append(0, *map(ctx.from_numpy, last))
    q = rand(rng, sum(new), nq * hd)
    got = attend(A, ctx, kv, 0, q)
    at = 0
    for i in ids:
        if new[i]:
            check(got[at:at + 1], q[at:at + 1], *(kv4_values(x[start[i]:start[i + 1]]) for x in (k, v)), nq, nkv, hd)
            at += 1
    pos = [rng.integers(0, x) for x in lens]  # more ranges than sequences: several launches
    ids2, pos2 = ids + ids, [int(p) for p in pos] * 2
    g = read(ctx, kv, 0, 1, ids2, pos2, [1] * len(ids2))
    for x, y in zip(g, (k, v)):
        same_bits(x, kv4_values(np.concatenate([y[start[i] + p:start[i] + p + 1] for i, p in zip(ids2, pos2)])))


# ------------------------------------------------------------------ pages

@pytest.mark.parametrize("seed", range(3))
def test_page_operations_keep_every_sequence(A, ctx, seed):
    """Random forks, copies, cuts, compactions and steps: every sequence reads back as its own history."""
    rng, pick = np.random.default_rng(seed), random.Random(seed)
    nq, nkv, hd, page, seqs, layers = 4, 2, 64, 32, 6, 3
    kv = A.KV4Cache(ctx, layers, nq, nkv, hd, 200, seqs, page, 24)
    have = {i: [np.empty((layers, 0, nkv * hd), np.float16)] * 2 for i in range(seqs)}
    for _ in range(60):
        op = pick.choice(["begin"] * 4 + ["fork", "copy", "truncate", "compact"])
        i, j = pick.randrange(seqs), pick.randrange(seqs)
        try:
            if op == "begin":
                ids = pick.sample(range(seqs), pick.randint(1, seqs))
                rows = [min(pick.choice([0, 1, 1, 5, 33]), 200 - kv.length(x)) for x in ids]
                kv.begin(ids, rows)
                k, v = (rand(rng, layers, sum(rows), nkv * hd) for _ in range(2))
                for l in range(layers):
                    kv.append(l, ctx.from_numpy(k[l]), ctx.from_numpy(v[l]))
                at = 0
                for x, r in zip(ids, rows):
                    have[x] = [np.concatenate([a, b[:, at:at + r]], 1) for a, b in zip(have[x], (k, v))]
                    at += r
                if sum(rows):
                    q = rand(rng, sum(rows), nq * hd)
                    got, at = attend(A, ctx, kv, 1, q), 0
                    for x, r in zip(ids, rows):
                        if r:
                            check(got[at:at + r], q[at:at + r], kv4_values(have[x][0][1]), kv4_values(have[x][1][1]), nq, nkv, hd)
                        at += r
            elif op == "truncate":
                n = pick.randint(0, kv.length(i))
                kv.truncate(i, n)
                have[i] = [x[:, :n] for x in have[i]]
            elif op == "compact":
                kv.compact()
            else:
                getattr(kv, op)(i, j)
                have[j] = list(have[i])
        except A.AesirError as e:
            assert e.code == -3 or "not empty" in str(e)
        lens = [kv.length(x) for x in range(seqs)]
        assert lens == [have[x][0].shape[1] for x in range(seqs)]
        if sum(lens):
            got = read(ctx, kv, 0, layers, list(range(seqs)), [0] * seqs, lens)
            for g, t in zip(got, (0, 1)):
                same_bits(g, kv4_values(np.concatenate([have[x][t] for x in range(seqs)], 1).reshape(-1, nkv * hd)))


def test_pages_past_four_gigabytes(A):
    """A pool of 5 GB: the rows of its last pages, their attention and their copies."""
    rng = np.random.default_rng(5)
    nq, nkv, hd, page = 8, 8, 128, 1024
    pages = (5 << 30) // (nkv * page * 160)
    need = A.KV4Cache.well_bytes(1, nq, nkv, hd, pages * page, 3, page, pages)
    with A.Context(need + (64 << 20)) as ctx:
        kv = A.KV4Cache(ctx, 1, nq, nkv, hd, pages * page, 3, page, pages)
        assert kv.page_bytes * pages > 1 << 32
        kv.begin([0], [(pages - 4) * page])  # positions without rows: only the table matters
        k, v, q = (rand(rng, 40, nkv * hd) for _ in range(3))
        kv.begin([1], [40])
        assert kv.pages(1) == [pages - 4]
        kv.append(0, ctx.from_numpy(k), ctx.from_numpy(v))
        check(attend(A, ctx, kv, 0, q), q, kv4_values(k), kv4_values(v), nq, nkv, hd)
        kv.copy(1, 2)
        for g, x in zip(read(ctx, kv, 0, 1, [2], [0], [40]), (k, v)):
            same_bits(g, kv4_values(x))
        kv.truncate(0, 0)
        assert kv.compact() == 2 and sorted(kv.pages(1) + kv.pages(2)) == [0, 1]
        for g, x in zip(read(ctx, kv, 0, 1, [1, 2], [0, 0], [40, 40]), (k, v)):
            same_bits(g, kv4_values(np.concatenate([x, x])))


def test_a_sequence_of_a_million_positions(A):
    """More table entries and page moves than one upload holds, and attention over 1.2 million positions: zeros (a
    fresh well) but for rows near the start, in the middle and at the end."""
    rng = np.random.default_rng(11)
    nq, nkv, hd, page, n = 4, 1, 32, 32, 1200000
    pages = -(-(n + 40) // page)
    with A.Context(A.KV4Cache.well_bytes(1, nq, nkv, hd, 2 * n, 3, page, 2 * pages) + (64 << 20)) as ctx:
        kv = A.KV4Cache(ctx, 1, nq, nkv, hd, 2 * n, 3, page, 2 * pages)
        K, V = np.zeros((2, n + 40, hd), np.float16)
        for start, rows in ((0, 50), (600000, 70), (n, 40)):
            if start > kv.length(0):
                kv.begin([0], [start - kv.length(0)])
            K[start:start + rows], V[start:start + rows] = rand(rng, rows, hd), rand(rng, rows, hd)
            K[start:start + rows] *= np.float16(3)
            kv.begin([0], [rows])
            kv.append(0, ctx.from_numpy(K[start:start + rows]), ctx.from_numpy(V[start:start + rows]))
        q = rand(rng, 40, nq * hd) * np.float16(2)
        got = attend(A, ctx, kv, 0, q)
        K, V = kv4_values(K), kv4_values(V)
        for r in (0, 39):
            check(got[r:r + 1], q[r:r + 1], K[:n + r + 1], V[:n + r + 1], nq, nkv, hd)
        kv.copy(0, 1)
        kv.truncate(0, 0)
        assert kv.compact() == pages and max(kv.pages(1)) == pages - 1
        kv.begin([1], [1])
        k, v = rand(rng, 1, hd), rand(rng, 1, hd)
        kv.append(0, ctx.from_numpy(k), ctx.from_numpy(v))
        got = attend(A, ctx, kv, 0, q[:1])
        check(got, q[:1], np.concatenate([K, kv4_values(k)]), np.concatenate([V, kv4_values(v)]), nq, nkv, hd)
        at, rows = [599990, n - 5, 0], [90, 46, 60]
        want = [np.concatenate([np.concatenate([x, kv4_values(y)])[a:a + b] for a, b in zip(at, rows)]) for x, y in ((K, k), (V, v))]
        for g, w in zip(read(ctx, kv, 0, 1, [1] * 3, at, rows), want):
            same_bits(g, w)


def test_a_merge_of_more_heads_and_rows_than_a_launch_holds(A):
    """A split row among prompts of 17 M rows and query heads in all."""
    rng = np.random.default_rng(13)
    nq, nkv, hd, page, prompts, rows, n = 64, 8, 32, 32, 4095, 65, 32768
    sizes = (1, nq, nkv, hd, n + page, prompts + 1, page, n // page + 1 + 3 * prompts)
    total = prompts * rows + 1
    assert total * nq > 1 << 24
    with A.Context(A.KV4Cache.well_bytes(*sizes) + 2 * total * (nq + nkv) * hd * 2 + (64 << 20)) as ctx:
        kv = A.KV4Cache(ctx, *sizes)
        K, V = np.zeros((2, n, nkv * hd), np.float16)  # a fresh well
        kv.begin([0], [n - 64])
        K[-64:], V[-64:] = rand(rng, 64, nkv * hd) * np.float16(3), rand(rng, 64, nkv * hd)
        kv.begin([0], [64])
        kv.append(0, ctx.from_numpy(K[-64:]), ctx.from_numpy(V[-64:]))
        # prompts repeat every 16 sequences
        k, v, q = (np.resize(rand(rng, 16 * rows, w * hd), (total, w * hd)) for w in (nkv, nkv, nq))
        kv.begin([*range(1, prompts + 1), 0], [rows] * prompts + [1])
        out = ctx.tensor(total, nq * hd)
        kv.append(0, ctx.from_numpy(k), ctx.from_numpy(v))
        kv.attention(0, ctx.from_numpy(q), out)
        got = out.numpy()
        have = [kv4_values(np.concatenate([a, b[-1:]])) for a, b in ((K, k), (V, v))]
        check(got[-1:].astype(np.float64), q[-1:], *have, nq, nkv, hd)
        for i in (0, 1000, prompts - 1):
            c = slice(i * rows, (i + 1) * rows)
            check(got[c].astype(np.float64), q[c], kv4_values(k[c]), kv4_values(v[c]), nq, nkv, hd)


# ------------------------------------------------------------------ capture, lifetimes, refusals

class Graph:
    """append and attention of one layer captured on the context's stream."""

    def __init__(self, A, ctx, calls):
        self.hip = C.CDLL("libamdhip64.so")
        self.stream, self.ctx = C.c_void_p(A._L.aesir_ctx_stream(ctx.h)), ctx
        graph, self.exec = C.c_void_p(), C.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 1) == 0  # thread-local
        try:
            calls()
        finally:
            rc = self.hip.hipStreamEndCapture(self.stream, C.byref(graph))
        assert rc == 0
        assert self.hip.hipGraphInstantiate(C.byref(self.exec), graph, None, None, C.c_size_t(0)) == 0
        assert self.hip.hipGraphDestroy(graph) == 0

    def launch(self):
        assert self.hip.hipGraphLaunch(self.exec, self.stream) == 0

    def close(self):
        self.ctx.synchronize()
        assert self.hip.hipGraphExecDestroy(self.exec) == 0


@pytest.mark.parametrize("rows", [1, 3])
def test_a_captured_step_serves_later_batches(A, ctx, rows):
    """One capture, many steps: lengths grow from one round past several splits, the order of sequences and
    their number change, a batch has more rows than the capture had, and none."""
    rng = np.random.default_rng(6)
    nq, nkv, hd, cap = 8, 2, 128, 6 * rows
    kv = A.KV4Cache(ctx, 1, nq, nkv, hd, 3000, 8, 64, 200)
    k, v, q = (ctx.tensor(cap, w * hd) for w in (nkv, nkv, nq))
    out = ctx.tensor(cap, nq * hd)
    have = {i: [np.empty((0, nkv * hd), np.float16)] * 2 for i in range(8)}
    ids = list(range(6))
    kv.begin(ids, [rows] * 6)
    kv.append(0, k, v)  # (the capture's batch is run once eagerly)
    kv.attention(0, q, out)
    g = Graph(A, ctx, lambda: (kv.append(0, k, v), kv.attention(0, q, out)))
    for i in range(6):
        kv.truncate(i, 0)
    out.upload(np.full((cap, nq * hd), 9.0, np.float16))
    g.launch()  # no batch: nothing is written
    assert (out.numpy() == 9.0).all()
    for step, (ids, news) in enumerate([(ids, [rows] * 6), ([5, 1, 3], [rows, 0, rows]), ([0, 7, 2, 4], [2 * rows, rows, rows, rows]),
                                        ([6, 0], [5 * rows, rows]), ([3], [4 * rows]), ([1, 2, 3, 4, 5, 6, 7], [rows] * 7)]):
        if step == 3:  # long earlier turns, so that work is split differently
            for i, n in ((6, 2500), (0, 700)):
                kk, vv = rand(rng, n, nkv * hd), rand(rng, n, nkv * hd)
                kv.begin([i], [n])
                kv.append(0, ctx.from_numpy(kk), ctx.from_numpy(vv))
                have[i] = [np.concatenate([a, b]) for a, b in zip(have[i], (kk, vv))]
        n = sum(news)
        x = [rand(rng, max(n, cap), w * hd) for w in (nkv, nkv, nq)]
        for t, y in zip((k, v, q), x):
            t.upload(y[:cap])
        kv.begin(ids, news)
        out.upload(np.full((cap, nq * hd), 9.0, np.float16))
        g.launch()
        got = out.numpy().astype(np.float64)
        at = 0
        for i, r in zip(ids, news):
            r_in = max(0, min(r, cap - at))  # rows past the capture's are not served
            have[i] = [np.concatenate([a, b[at:at + r]]) for a, b in zip(have[i], x)]
            if r and r_in == r:
                check(got[at:at + r], x[2][at:at + r], *map(kv4_values, have[i]), nq, nkv, hd)
            at += r
        assert (got[n:] == 9.0).all()
        if n > cap:  # finish the batch eagerly
            kv.append(0, ctx.from_numpy(x[0]), ctx.from_numpy(x[1]))
        got2 = attend(A, ctx, kv, 0, x[2][:n])  # (a launch of this batch's own shape: other orders of sums)
        at = 0
        for i, r in zip(ids, news):
            if r:
                check(got2[at:at + r], x[2][at:at + r], *map(kv4_values, have[i]), nq, nkv, hd)
            at += r
    g.close()


def test_a_capture_of_many_sequences_serves_long_ones(A):
    """A grid of 4096 workgroups a KV head, replayed for 4096 forks of a long sequence: 700 K rounds to a workgroup, so the
    starts of those that have no work lie past 32 bits."""
    rng = np.random.default_rng(12)
    nkv, hd, page, seqs, n = 256, 32, 32, 4096, 16384
    sizes = (1, nkv, nkv, hd, n + page, seqs, page, n // page + seqs)
    with A.Context(A.KV4Cache.well_bytes(*sizes) + (512 << 20)) as ctx:
        kv = A.KV4Cache(ctx, *sizes)
        ids, new = list(range(seqs)), [1] * seqs
        k, v, q, out = (ctx.tensor(seqs, nkv * hd) for _ in range(4))
        kv.begin(ids, new)
        g = Graph(A, ctx, lambda: (kv.append(0, k, v), kv.attention(0, q, out)))
        for i in ids:
            kv.truncate(i, 0)
        K, V = np.zeros((2, n, nkv * hd), np.float16)  # a fresh well
        kv.begin([0], [n - 64])
        K[-64:], V[-64:] = rand(rng, 64, nkv * hd) * np.float16(3), rand(rng, 64, nkv * hd)
        kv.begin([0], [64])
        kv.append(0, ctx.from_numpy(K[-64:]), ctx.from_numpy(V[-64:]))
        for i in ids[1:]:
            kv.fork(0, i)
        x = [rand(rng, seqs, nkv * hd) for _ in range(3)]
        for t, y in zip((k, v, q), x):
            t.upload(y)
        kv.begin(ids, new)
        for _ in range(2):
            out.upload(np.full((seqs, nkv * hd), 9.0, np.float16))
            g.launch()
            got = out.numpy().astype(np.float64)
            for r in (0, 1365, 1366, 4095):
                for h in (0, 100, 255):
                    c = slice(h * hd, (h + 1) * hd)
                    have = [kv4_values(np.concatenate([a[:, c], b[r:r + 1, c]])) for a, b in zip((K, V), x)]
                    check(got[r:r + 1, c], x[2][r:r + 1, c], *have, 1, 1, hd)
        g.close()


def test_changes_are_refused_while_capturing(A, ctx):
    kv = A.KV4Cache(ctx, 1, 2, 1, 64, 64, 3, 32, 4)
    t = ctx.tensor(1, 128)
    kv.begin([0], [1])
    calls = [lambda: kv.begin([1], [1]), lambda: kv.fork(0, 1), lambda: kv.copy(0, 1), lambda: kv.truncate(0, 0), kv.compact,
             lambda: kv.read(0, 1, [0], [0], [1], t, t)]
    calls.append(lambda: A.KV4Cache(ctx, 1, 2, 1, 64, 64, 3, 32, 4))
    refused = []

    def run():
        for call in calls:
            try:
                call()
            except A.AesirError as e:
                refused.append("captured" in str(e))
        kv.append(0, t, t)

    g = Graph(A, ctx, run)
    assert refused == [True] * len(calls) and kv.length(0) == 1 and kv.free_pages == 3
    g.close()


def test_destroy_waits_for_the_end_of_a_capture(A, ctx):
    kv, other = (A.KV4Cache(ctx, 1, 2, 1, 64, 64, 3, 32, 4) for _ in range(2))
    t = ctx.tensor(1, 128)
    kv.begin([0], [1])

    def run():
        with pytest.raises(A.AesirError, match="captured"):
            other.close()
        kv.append(0, t, t)

    Graph(A, ctx, run).close()
    other.close()
    assert other.h is None


def test_refusals(A, ctx):
    kv = A.KV4Cache(ctx, 2, 4, 2, 64, 64, 3, 32, 6)
    k, q = ctx.tensor(3, 128), ctx.tensor(3, 256)
    none = A.Tensor(ctx, None, 3, 256)
    for call in (lambda: kv.append(0, k, k), lambda: kv.attention(0, q, q)):
        with pytest.raises(A.AesirError, match="no batch"):
            call()
    kv.begin([0, 1], [2, 1])
    thin, short = ctx.tensor(3, 100), ctx.tensor(2, 256)
    odd = A.Tensor(ctx, k.ptr + 1, 3, 128)
    for call, text in [(lambda: kv.append(2, k, k), "layer"), (lambda: kv.append(-1, k, k), "layer"), (lambda: kv.attention(2, q, q), "layer"),
                       (lambda: kv.append(0, short, k), "3 new rows"), (lambda: kv.append(0, k, short), "3 new rows"),
                       (lambda: kv.append(0, thin, k), "narrower"), (lambda: kv.append(0, k, thin), "narrower"), (lambda: kv.append(0, none, k), "null"),
                       (lambda: kv.attention(0, short, q), "3 new rows"), (lambda: kv.attention(0, q, short), "3 new rows"),
                       (lambda: kv.attention(0, k, q), "narrower"), (lambda: kv.attention(0, q, k), "narrower"), (lambda: kv.attention(0, q, none), "null"),
                       (lambda: kv.append(0, odd, k), "2-byte"), (lambda: kv.attention(0, q, A.Tensor(ctx, q.ptr + 1, 3, 256)), "2-byte"),
                       (lambda: kv.read(0, 1, [0, 1], [0, 0], [2, 1], k, odd), "2-byte"),
                       (lambda: kv.read(0, 3, [0], [0], [1], k, k), "layer"), (lambda: kv.read(1, 2, [0], [0], [1], k, k), "layer"),
                       (lambda: kv.read(0, 1, [3], [0], [1], k, k), "not in"), (lambda: kv.read(0, 1, [0], [1], [2], k, k), "outside"),
                       (lambda: kv.read(0, 1, [0], [-1], [1], k, k), "outside"), (lambda: kv.read(0, 1, [0], [0], [2], k, k), "2 rows"),
                       (lambda: kv.read(0, 1, [0, 1], [0, 0], [2, 1], thin, k), "narrower"), (lambda: kv.read(0, 1, [0, 1], [0, 0], [2, 1], none, k), "null")]:
        with pytest.raises(A.AesirError, match=text):
            call()
    kv.begin([2], [0])  # a batch without rows: the calls have nothing to do
    zero = A.Tensor(ctx, None, 0, 0)
    kv.append(0, zero, zero)
    kv.attention(0, zero, zero)
    kv.read(0, 2, [2], [0], [0], zero, zero)
    for end in (lambda: kv.fork(0, 2), lambda: kv.truncate(2, 0), lambda: kv.copy(0, 2), kv.compact):
        kv.begin([0], [1])
        end()
        with pytest.raises(A.AesirError, match="no batch"):
            kv.append(0, k.view(1, 128), k.view(1, 128))


def test_lifetimes(A):
    """The context outlives its caches; a well without room refuses one and keeps its offset; two caches of one
    context do not meet; a cache on used memory starts without a batch."""
    rng = np.random.default_rng(8)
    ctx = A.Context(64 << 20)
    with pytest.raises(A.AesirError) as e:
        A.KV4Cache(ctx, 32, 8, 8, 128, 4096, 4, 64, 256)
    assert e.value.code == -3 and ctx.offset == 0
    junk = ctx.from_numpy(np.full((1, 1 << 20), np.nan, np.float16))
    junk.upload(rng.integers(0, 1 << 15, (1, 1 << 20)).astype(np.uint16).view(np.float16))
    ctx.synchronize()
    ctx.reset(0)
    a, b = (A.KV4Cache(ctx, 1, 2, 1, 64, 100, 2, 32, 8) for _ in range(2))
    assert A._L.aesir_ctx_destroy(ctx.h) == -1 and "alive" in A.last_error()
    xs = [[rand(rng, 50, 64), rand(rng, 50, 64)] for _ in range(2)]
    for kv, x in zip((a, b), xs):
        kv.begin([1], [50])
        kv.append(0, *map(ctx.from_numpy, x))
    q = rand(rng, 50, 128)
    for kv, x in zip((a, b), xs):
        check(attend(A, ctx, kv, 0, q), q, *map(kv4_values, x), 2, 1, 64)
    a.close()
    for g, x in zip(read(ctx, b, 0, 1, [1], [0], [50]), xs[1]):
        same_bits(g, kv4_values(x))
    ctx.close()  # closes b first
    assert b.h is None


# ------------------------------------------------------------------ weights

def half_weights(hd, q_rows, heads):
    """Query rows whose score against a key of ones is d above that of a key of zeros, e^-d = (1 + 2^-11 + 2^-13) / 2: a weight
    that f16 rounds up by 2^-11 - 2^-13 of itself."""
    total = -np.log(0.5 * (1 + 2.0 ** -11 + 2.0 ** -13)) * np.sqrt(hd)
    q = np.full(hd, total / hd).astype(np.float16)
    q[0] = np.float16(float(q[0]) + total - q.astype(np.float64).sum())
    got = 2 * np.exp(-q.astype(np.float64).sum() / np.sqrt(hd)) - 1
    assert 2.0 ** -11 + 2.0 ** -14 < got < 2.0 ** -10
    return np.tile(q, (q_rows, heads))


@pytest.mark.parametrize("hd,nq,nkv,length,rows", [(128, 4, 1, 4096, 1), (64, 32, 8, 8192, 8), (64, 32, 8, 8192, 16), (32, 32, 8, 8192, 128),
                                                   (64, 32, 8, 8192, 128), (128, 32, 8, 8192, 128), (256, 4, 4, 2000, 1), (256, 16, 4, 4096, 64)])
@pytest.mark.parametrize("value", [65504.0, -65504.0, 1.5])
def test_weights_sum_to_one(A, ctx, hd, nq, nkv, length, rows, value):
    """Equal values come out as they are, the largest f16 among them, where 31 of 32 weights round the same way (each wave
    meets a key of weight one in each round of 32, so that its maximum is that key's). A lane's
    chain of sums is at most 8192 / 4 / 2 dot products of 3 * 2^-24 (and 256 matrix instructions of 2^-23): 2.2e-4 of the
    weights' sum, under half an f16 step (2.4e-4)."""
    kv = A.KV4Cache(ctx, 1, nq, nkv, hd, length, 1, 64, -(-length // 64))
    k, v = np.zeros((length, nkv * hd), np.float16), np.full((length, nkv * hd), value, np.float16)
    k[::32] = 1
    mark = ctx.offset
    if length > rows:
        kv.begin([0], [length - rows])
        kv.append(0, ctx.from_numpy(k[:-rows]), ctx.from_numpy(v[:-rows]))
        ctx.reset(mark)
    kv.begin([0], [rows])
    kv.append(0, ctx.from_numpy(k[-rows:]), ctx.from_numpy(v[-rows:]))
    got = attend(A, ctx, kv, 0, half_weights(hd, rows, nq))
    assert (got == value).all(), (got[got != value][:5], (got != value).sum())


def test_a_cache_dropped_during_a_capture_does_not_outlive_its_context(A):
    ctx = A.Context(64 << 20)
    caches = [A.KV4Cache(ctx, 1, 2, 1, 64, 64, 3, 32, 4) for _ in range(2)]
    t = ctx.tensor(1, 128)
    caches[0].begin([0], [1])

    def run():
        caches.pop()
        caches[0].append(0, t, t)

    Graph(A, ctx, run).close()
    ctx.close()
    assert not ctx.h and not caches[0].h
