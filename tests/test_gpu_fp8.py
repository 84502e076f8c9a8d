"""The 8-bit floating-point operators through the C ABI against their definitions in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from fp8_tools import NUMBERS, nearest, quantize, same_codes, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A():
    import aesir_hip

    return aesir_hip


@pytest.fixture(scope="module")
def ctx(A):
    with A.Context(1 << 30) as c:
        yield c


@pytest.fixture(autouse=True)
def well(request):
    if "ctx" in request.fixturenames:
        c = request.getfixturevalue("ctx")
        mark = c.offset
        yield
        c.reset(mark)
    else:
        yield


def put(A, ctx, a, stride=None, shift=0):
    """a on the device in rows `stride` elements apart, `shift` elements off the well's alignment."""
    rows, cols = a.shape
    stride = stride or cols
    room = np.full((rows, stride), np.nan, np.float16)
    room[:, :cols] = a
    t = ctx.tensor(1, rows * stride + shift)
    return A.Tensor(ctx, t.ptr + 2 * shift, rows, stride).upload(room)


def dirty(A, ctx, rows, cols, block_rows=1):
    """An 8-bit matrix whose room holds other bytes."""
    t = A.FP8Tensor.empty(ctx, rows, cols, block_rows)
    return t.upload(np.full((rows, t.ld), 0x55, np.uint8), np.full(t.scales_shape, 7.0, np.float32))


def check(t, codes, scales, eps):
    got = t.scales().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(scales))
    fine = ~np.isnan(scales)
    assert np.all(np.abs(got - scales)[fine] <= eps * scales[fine]), np.max(np.abs(got - scales)[fine] / np.maximum(scales[fine], 1e-300))
    assert same_codes(t.codes(), codes)


def activations(rng, rows, cols):
    """Rows with a few strong channels, zeros, a block of zeros and the smallest numbers among them."""
    x = rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal(cols))
    x[:, :: max(1, cols // 5)] *= 30
    x[rng.random((rows, cols)) < 0.05] = 0
    x = x.astype(np.float16)
    x[rows // 2, : min(cols, 128)] = 0
    x[0, -min(cols, 40):] = np.float16(6e-8) * np.arange(min(cols, 40))
    return x


# ------------------------------------------------------------------ quantize

@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols,stride,shift", [(1, 1, None, 0), (1, 128, None, 0), (3, 127, 160, 0), (7, 129, None, 3), (2, 304, 304, 0),
                                                    (130, 256, 264, 0), (257, 1000, None, 0), (128, 8, None, 0), (129, 520, 1040, 1), (5, 16392, None, 0)])
def test_quantize(A, ctx, rows, cols, stride, shift, block_rows):
    x = activations(np.random.default_rng(rows * cols), rows, cols)
    t = dirty(A, ctx, rows, cols, block_rows)
    A.quantize_fp8(ctx, put(A, ctx, x, stride, shift), t)
    # the scale is one correctly rounded quotient
    check(t, *quantize(x.astype(np.float64), block_rows), 2.0**-24)
    assert np.array_equal(t.numpy(), values(t.codes(), t.scales(), block_rows).astype(np.float32)[:, :cols])


@pytest.mark.parametrize("top", [65504.0, 448.0, 449.0, 1.0, 7.0, 0.3, 6.1e-5, 6e-8])
def test_every_f16_beside_a_largest_value(A, ctx, top):
    """All f16 numbers up to `top`, 127 a block: ties (many at 448 and 7 times a power of two), e4m3's smallest
    numbers and f16's among them."""
    top = np.float16(top)
    all16 = np.arange(65536, dtype=np.uint32).astype(np.uint16).view(np.float16)
    v = all16[np.abs(all16) <= top]
    x = np.zeros((-(-len(v) // 127), 128), np.float16)
    x[:, 1:].reshape(-1)[: len(v)] = 0
    flat = np.zeros(x.shape[0] * 127, np.float16)
    flat[: len(v)] = v
    x[:, 0], x[:, 1:] = top, flat.reshape(-1, 127)
    t = dirty(A, ctx, *x.shape)
    A.quantize_fp8(ctx, put(A, ctx, x), t)
    codes, scales = quantize(x.astype(np.float64))
    check(t, codes, scales, 2.0**-24)
    assert np.array_equal(t.codes() & 127, codes & 127)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_inf_and_nan(A, ctx, bad, block_rows):
    x = np.random.default_rng(1).standard_normal((200, 400)).astype(np.float16)
    x[3, 200] = x[150, 399] = bad
    t = dirty(A, ctx, 200, 400, block_rows)
    A.quantize_fp8(ctx, put(A, ctx, x), t)
    check(t, *quantize(x.astype(np.float64), block_rows), 2.0**-24)


# ------------------------------------------------------------------ RMSNorm

def norm64(x, residual, w, eps):
    with np.errstate(all="ignore"):
        h = x if residual is None else (x.astype(np.float64) + residual).astype(np.float16)
        p = h.astype(np.float64) * w.astype(np.float64)
        p[~np.isfinite(h).all(1)] = np.nan
        codes, scales = quantize(p)
        return h, codes, scales / np.sqrt((h.astype(np.float64) ** 2).mean(1) + eps)


def norm_eps(cols):
    """A thread's sum of 8 squares for each 2048 columns, the wave's and the workgroup's 10 steps, half of it behind the
    root; the mean's quotient and sum, half of them too, and root, quotient, product and quotient: a rounding each."""
    return ((8 * -(-cols // 2048) + 12) / 2 + 4) * 2.0**-24


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols,stride,shift", [(1, 1, None, 0), (1, 2048, None, 0), (4, 64, None, 0), (3, 127, 131, 1), (33, 1001, None, 0),
                                                    (65, 4096, 4104, 0), (2, 8200, None, 0), (5, 14336, None, 0), (1, 40000, None, 0), (300, 288, 576, 0)])
def test_norm(A, ctx, rows, cols, stride, shift, residual):
    rng = np.random.default_rng(cols + rows)
    x = activations(rng, rows, cols)
    w = (1 + 0.3 * rng.standard_normal((1, cols))).astype(np.float16)
    r = (rng.standard_normal((rows, cols)) * 0.3).astype(np.float16) if residual else None
    t, tx = dirty(A, ctx, rows, cols), put(A, ctx, x, stride, shift)
    h, codes, scales = norm64(x, r, w, 1e-5)
    if residual:
        total = put(A, ctx, np.zeros_like(x), stride, shift)
        A.rmsnorm_fp8(ctx, tx, put(A, ctx, w), t, 1e-5, put(A, ctx, r, cols + 16), total)
        assert np.array_equal(total.numpy()[:, :cols].view(np.uint16), h.view(np.uint16))
        assert np.isnan(total.numpy()[:, cols:]).all()
    else:
        A.rmsnorm_fp8(ctx, tx, put(A, ctx, w), t, 1e-5)
    assert np.array_equal(tx.numpy()[:, :cols].view(np.uint16), x.view(np.uint16))
    check(t, codes, scales, norm_eps(cols))


@pytest.mark.parametrize("into", ["x", "residual"])
@pytest.mark.parametrize("cols", [96, 131, 2048, 20000])
def test_norm_in_place(A, ctx, into, cols):
    rng = np.random.default_rng(cols)
    x, r = activations(rng, 6, cols), activations(rng, 6, cols)
    w = rng.standard_normal((1, cols)).astype(np.float16)
    tx, tr, t = put(A, ctx, x), put(A, ctx, r), dirty(A, ctx, 6, cols)
    A.rmsnorm_fp8(ctx, tx, put(A, ctx, w), t, 1e-6, tr, tx if into == "x" else tr)
    h, codes, scales = norm64(x, r, w, 1e-6)
    assert np.array_equal((tx if into == "x" else tr).numpy().view(np.uint16), h.view(np.uint16))
    assert np.array_equal((tr if into == "x" else tx).numpy().view(np.uint16), (r if into == "x" else x).view(np.uint16))
    check(t, codes, scales, norm_eps(cols))


@pytest.mark.parametrize("cols", [300, 4096, 20000])
def test_norm_inf_nan_and_zeros(A, ctx, cols):
    """A row with an inf, a NaN or a sum past f16 is NaN whole; an inf in the weight makes one block NaN; zeros stay."""
    rng = np.random.default_rng(5)
    x, r = (rng.standard_normal((6, cols)).astype(np.float16) for _ in range(2))
    w = rng.standard_normal((1, cols)).astype(np.float16)
    x[0, 7], x[1, cols - 1], x[2, 130], r[2, 130] = np.nan, -np.inf, 65504, 65504
    x[3], r[3] = 0, 0
    x[4, 256:], r[4, 256:] = 0, 0
    w[0, 5] = np.inf
    t, total = dirty(A, ctx, 6, cols), put(A, ctx, x)
    A.rmsnorm_fp8(ctx, put(A, ctx, x), put(A, ctx, w), t, 1e-5, put(A, ctx, r), total)
    h, codes, scales = norm64(x, r, w, 1e-5)
    assert np.isnan(scales[:, :3]).all() and np.isnan(scales[0]).all() and not np.isnan(scales[1:, 3:]).any()
    assert np.array_equal(total.numpy(), h, equal_nan=True)
    check(t, codes, scales, norm_eps(cols))


def test_norm_of_f16_least_and_largest(A, ctx):
    """Squares past f16 and under f32's usual range of activations; the factor is 1 / sqrt(eps) or the row's."""
    x = np.concatenate([np.full((1, 640), 6e-8), np.full((1, 640), 65504.0), np.tile([6e-8, -1e-7], (1, 320))]).astype(np.float16)
    w = np.linspace(-3, 65504, 640).astype(np.float16)[None]
    for eps in (1e-5, 1e-14):
        t = dirty(A, ctx, 3, 640)
        A.rmsnorm_fp8(ctx, put(A, ctx, x), put(A, ctx, w), t, eps)
        # epsilon is an f32
        check(t, *norm64(x, None, w, float(np.float32(eps)))[1:], norm_eps(640))


# ------------------------------------------------------------------ SwiGLU

def swiglu64(g, u):
    with np.errstate(all="ignore"):
        g, u = g.astype(np.float64), u.astype(np.float64)
        y = u * g / (1 + np.exp(-g))
        y[~(np.isfinite(g) & np.isfinite(u))] = np.nan
    return quantize(y, least=2.0**-64)


# the values are at most 4 units of f32's last place (2^-23) off, the quotient half a one more
SWIGLU_EPS = 4.5 * 2.0**-23


@pytest.mark.parametrize("rows,cols,fused,shift", [(1, 1, False, 0), (1, 5632, True, 0), (3, 127, True, 0), (64, 172, True, 0), (65, 1001, False, 1),
                                                   (200, 14336, True, 0), (17, 256, False, 0)])
def test_swiglu(A, ctx, rows, cols, fused, shift):
    rng = np.random.default_rng(rows + cols)
    g, u = activations(rng, rows, cols), activations(rng, rows, cols)
    t = dirty(A, ctx, rows, cols)
    if fused:
        both = put(A, ctx, np.concatenate([g, u], 1), None, shift)
        tg, tu = A.Tensor(ctx, both.ptr, rows, 2 * cols), A.Tensor(ctx, both.ptr + 2 * cols, rows, 2 * cols)
    else:
        tg, tu = put(A, ctx, g, None, shift), put(A, ctx, u, cols + 8)
    A.swiglu_fp8(ctx, tg, tu, t)
    check(t, *swiglu64(g, u), SWIGLU_EPS)


def test_swiglu_far_gates(A, ctx):
    """Every f16 gate: exponentials past f32 either way, blocks whose values are all next to nothing, inf and NaN."""
    all16 = np.arange(65536, dtype=np.uint32).astype(np.uint16).view(np.float16)
    g = np.sort(all16[~np.isnan(all16)])
    g = np.concatenate([g, np.full(-len(g) % 1024 + 1, 5), np.full(1023, np.nan)]).astype(np.float16).reshape(-1, 1024)
    for scale in (1.0, 6e-8, 65504.0):
        u = np.full_like(g, scale)
        t = dirty(A, ctx, *g.shape)
        A.swiglu_fp8(ctx, put(A, ctx, g), put(A, ctx, u), t)
        check(t, *swiglu64(g, u), SWIGLU_EPS)


@pytest.mark.parametrize("lowest", [-46, -52])
def test_swiglu_next_to_the_least_block(A, ctx, lowest):
    """Blocks whose largest value is just above 2^-64, and from -52 on below it too."""
    g = np.linspace(lowest, -38, 128 * 64).astype(np.float16).reshape(64, 128)
    u = np.linspace(0.5, 2, 128 * 64).astype(np.float16).reshape(64, 128)
    t = dirty(A, ctx, 64, 128)
    A.swiglu_fp8(ctx, put(A, ctx, g), put(A, ctx, u), t)
    codes, scales = swiglu64(g, u)
    assert (scales > 0).any() and (scales == 0).any() == (lowest == -52)
    check(t, codes, scales, SWIGLU_EPS)


@pytest.mark.parametrize("where", ["gate", "up"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_swiglu_inf_and_nan(A, ctx, where, bad):
    rng = np.random.default_rng(2)
    g, u = (rng.standard_normal((5, 384)).astype(np.float16) for _ in range(2))
    (g if where == "gate" else u)[2, 140] = bad
    (u if where == "gate" else g)[2, 140] = 0
    t = dirty(A, ctx, 5, 384)
    A.swiglu_fp8(ctx, put(A, ctx, g), put(A, ctx, u), t)
    check(t, *swiglu64(g, u), SWIGLU_EPS)


# ------------------------------------------------------------------ product

def matrix(A, ctx, codes, scales, cols, block_rows):
    return A.FP8Tensor.empty(ctx, len(codes), cols, block_rows).upload(codes, scales)


def random_matrix(rng, rows, cols, block_rows):
    """Codes of all finite numbers and scales over a few powers of two, zeros behind cols."""
    nb = -(-cols // 128)
    codes = rng.integers(0, 127, (rows, nb * 128)).astype(np.uint8) | (rng.integers(0, 2, (rows, nb * 128)) << 7).astype(np.uint8)
    codes[:, cols:] = 0
    shape = (nb, rows) if block_rows == 1 else (-(-rows // 128), nb)
    return codes, np.exp2(rng.uniform(-9, -5, shape)).astype(np.float32)


def product(A, ctx, a, b, cols, f32, extra=0):
    M, N = len(a[0]), len(b[0])
    dtype = np.float32 if f32 else np.float16
    c = ctx.tensor(M, N + extra, dtype).upload(np.full((M, N + extra), -77.0))
    A.gemm_fp8(ctx, matrix(A, ctx, *a, cols, 1), matrix(A, ctx, *b, cols, 128), A.Tensor(ctx, c.ptr, M, N + extra, dtype))
    out = c.numpy()
    assert np.all(out[:, N:] == -77.0)
    return out[:, :N]


def assert_near(got, a, b, f32):
    """Every addition along k is at most a unit of f32's last place off, whichever way the matrix cores round, every
    block's scale and product half a one each; then half a step of the output's type (f16's least is 2^-24).

    f16 results may come from the 8-bit matrix instructions, which line up the products of 8 neighbouring k at the
    largest's power of two, 2^e, and drop what lies under 2^(e - 13): at most that much of each of the 8, and the
    largest product is 2^e or more."""
    x, w = values(*a), values(*b, 128)
    want, mass = x @ w.T, np.abs(x) @ np.abs(w).T
    bound = mass * (x.shape[1] + 8) * 2.0**-23
    if not f32:
        for k in range(0, x.shape[1], 8):
            bound += 8 * 2.0**-13 * (np.abs(x[:, None, k:k + 8]) * np.abs(w[None, :, k:k + 8])).max(2) if len(x) * len(w) <= 1 << 16 else \
                2.0**-10 * np.abs(x[:, k:k + 8]).max(1)[:, None] * np.abs(w[:, k:k + 8]).max(1)
        bound += np.abs(want) * 2.0**-11 + 2.0**-25
    off = np.abs(got.astype(np.float64) - want)
    assert np.all(off <= bound), (np.argwhere(~(off <= bound))[:4], np.max(off / bound))


SIZES = [(1, 1, 1), (1, 128, 128), (1, 16, 4096), (1, 300, 2048), (1, 6144, 1000), (2, 129, 127), (3, 1000, 1024), (15, 16, 129), (16, 100, 256),
         (17, 257, 640), (16, 2000, 384), (31, 64, 5632), (33, 2048, 300), (48, 15, 64), (63, 500, 1408), (64, 1030, 2048), (65, 128, 172), (100, 3000, 512),
         (127, 127, 127), (128, 128, 128), (129, 385, 1152), (200, 1111, 999), (256, 256, 8192), (333, 2048, 768), (511, 100, 2048),
         (1025, 640, 256), (700, 5000, 512)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(A, ctx, M, N, K):
    rng = np.random.default_rng(M * 7 + N * 3 + K)
    a, b = random_matrix(rng, M, K, 1), random_matrix(rng, N, K, 128)
    assert_near(product(A, ctx, a, b, K, True, 3), a, b, True)
    a = (a[0], a[1] * 2.0**-6)  # within f16
    assert_near(product(A, ctx, a, b, K, False), a, b, False)
    assert_near(product(A, ctx, a, b, K, False, 5), a, b, False)


@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_of_whole_numbers(A, ctx, M, N, K):
    """Small whole numbers and scales that are powers of two: every sum is exact, so is the result."""
    rng = np.random.default_rng(M + N + K)
    ones = nearest(np.arange(-2.0, 3.0))
    a, b = random_matrix(rng, M, K, 1), random_matrix(rng, N, K, 128)
    for codes, scales in (a, b):
        codes[:, :K] = ones[rng.integers(0, 5, (len(codes), K))]
        scales[:] = np.exp2(rng.integers(-1, 2, scales.shape))
    got = product(A, ctx, a, b, K, True)
    assert np.array_equal(got, (values(*a) @ values(*b, 128).T).astype(np.float32))


@pytest.mark.parametrize("M", [1, 9, 40, 70, 300, 2000])
def test_every_code(A, ctx, M):
    """Each code alone in its row, times one: every product is that number, in both types."""
    rows = np.arange(M)
    codes, scales = np.zeros((M, 384), np.uint8), np.ones((3, M), np.float32)
    ones = np.full((256, 384), nearest(np.array([1.0]))[0], np.uint8)
    for first in range(0, 256, 128 if M < 256 else 256):
        codes[:] = 0
        c = (first + rows) % 256
        c = np.where(c & 127 == 127, 0, c).astype(np.uint8)
        codes[rows, (7 * rows) % 384] = c
        for f32 in (True, False):
            got = product(A, ctx, (codes, scales), (ones, np.ones((2, 3), np.float32)), 384, f32)
            assert np.array_equal(got, np.repeat(NUMBERS[c][:, None], 256, 1).astype(got.dtype))


@pytest.mark.parametrize("M,N", [(1, 40), (20, 40), (40, 130), (70, 130)])
def test_long_rows(A, ctx, M, N):
    """A quarter of a million columns of whole numbers: exact sums, in stretches too."""
    K = (1 << 18) - 5
    rng = np.random.default_rng(M)
    ones = nearest(np.arange(-2.0, 3.0))
    values8 = [rng.integers(0, 5, (n, K)) for n in (M, N)]
    nb = -(-K // 128)
    a, b = (np.zeros((n, nb * 128), np.uint8) for n in (M, N))
    a[:, :K], b[:, :K] = ones[values8[0]], ones[values8[1]]
    got = product(A, ctx, (a, np.ones((nb, M), np.float32)), (b, np.ones((-(-N // 128), nb), np.float32)), K, True)
    assert np.array_equal(got, (values8[0] - 2.0).astype(np.float32) @ (values8[1] - 2.0).T.astype(np.float32))


@pytest.mark.parametrize("M,N,K", [(1, 300, 512), (20, 300, 512), (64, 500, 384), (150, 300, 640), (520, 700, 256)])
def test_product_nan_stays_in_its_rows(A, ctx, M, N, K):
    """A NaN code or scale reaches its row of A or its rows of B, and nothing else."""
    rng = np.random.default_rng(9)
    a, b = random_matrix(rng, M, K, 1), random_matrix(rng, N, K, 128)
    want = values(*a) @ values(*b, 128).T
    a[0][M // 2, 200], b[0][131, 100], b[1][2, 1] = 0x7F, 0xFF, np.nan
    got = product(A, ctx, a, b, K, True)
    nan = np.zeros((M, N), bool)
    nan[M // 2], nan[:, 131], nan[:, 256:384] = True, True, True
    assert np.array_equal(np.isnan(got), nan)
    assert np.allclose(got[~nan], want[~nan], rtol=1e-3, atol=1e-3 * np.abs(want).max())


def test_product_past_f16_is_inf(A, ctx):
    a, b = random_matrix(np.random.default_rng(1), 3, 128, 1), random_matrix(np.random.default_rng(2), 20, 128, 128)
    a[0][:], b[0][:] = nearest(np.array([448.0])), nearest(np.array([-448.0]))
    a[1][:], b[1][:] = 1, 1
    assert np.all(np.isneginf(product(A, ctx, a, b, 128, False)))
    assert np.all(product(A, ctx, a, b, 128, True) == -(448.0**2) * 128)


def test_same_call_same_bits(A, ctx):
    rng = np.random.default_rng(11)
    for M, N, K in ((1, 6144, 4096), (64, 1000, 5632), (300, 1000, 2048)):
        a, b = random_matrix(rng, M, K, 1), random_matrix(rng, N, K, 128)
        first = product(A, ctx, a, b, K, True)
        for _ in range(3):
            assert np.array_equal(product(A, ctx, a, b, K, True).view(np.uint32), first.view(np.uint32))


def test_offsets_past_32_bits(A):
    """Rows whose elements and codes lie past 2^32 bytes: the last ones of 1.1 million rows of 4096."""
    rows, cols, last = 1_100_000, 4096, 300
    rng = np.random.default_rng(3)
    x = rng.standard_normal((last, cols)).astype(np.float16)
    w = random_matrix(rng, 40, cols, 128)
    with A.Context(15 << 30) as ctx:
        t, tx = A.FP8Tensor.empty(ctx, rows, cols), ctx.tensor(rows, cols)
        c = ctx.tensor(rows, 40, np.float32)
        tx.view(last, cols, (rows - last) * cols).upload(x)
        A.quantize_fp8(ctx, tx, t)
        A.gemm_fp8(ctx, t, matrix(A, ctx, *w, cols, 128), c)
        codes, scales = quantize(x.astype(np.float64))
        got = A.Tensor(ctx, t.ptr + (rows - last) * cols, last, cols, np.uint8).numpy()
        assert same_codes(got, codes)
        assert_near(c.view(last, 40, (rows - last) * 40).numpy(), (codes, t.scales()[:, -last:]), w, True)
        assert np.all(c.view(last, 40).numpy() == 0)
        A.rmsnorm_fp8(ctx, tx, ctx.from_numpy(np.ones(cols)), t)
        assert same_codes(A.Tensor(ctx, t.ptr + (rows - last) * cols, last, cols, np.uint8).numpy(), codes)
        A.swiglu_fp8(ctx, tx, tx, t)
        assert same_codes(A.Tensor(ctx, t.ptr + (rows - last) * cols, last, cols, np.uint8).numpy(), swiglu64(x, x)[0])


@pytest.mark.parametrize("rows,cols", [((1 << 23) + 1000, 40), (16387, 2100)])
def test_many_rows(A, rows, cols):
    """The row calls past 2^23 rows, more than a launch takes, and of 2^18 blocks or more of long rows: first, last and
    middle rows, whose scales lie far apart."""
    rng = np.random.default_rng(8)
    x = rng.standard_normal((rows, cols), dtype=np.float32).astype(np.float16)
    at = np.r_[0:50, rows - 1050:rows - 950, rows - 50:rows]
    w = rng.standard_normal(cols).astype(np.float16)
    with A.Context(4 << 30) as ctx:
        t, tx, tw = A.FP8Tensor.empty(ctx, rows, cols), ctx.from_numpy(x), ctx.from_numpy(w)
        for call, want in ((lambda: A.quantize_fp8(ctx, tx, t), quantize(x[at].astype(np.float64))), (lambda: A.swiglu_fp8(ctx, tx, tx, t), swiglu64(x[at], x[at])),
                           (lambda: A.rmsnorm_fp8(ctx, tx, tw, t), norm64(x[at], None, w[None], 1e-5)[1:])):
            call()
            assert same_codes(t.codes()[at], want[0])
            assert np.allclose(t.scales()[:, at], want[1], rtol=1e-6, atol=0)


# ------------------------------------------------------------------ a layer's MLP

class Mlp:
    """The second half of a Llama layer in 8 bits: norm with the residual, gate and up rows, SwiGLU, down, residual."""

    def __init__(self, A, ctx, rows, dim, ffn, seed):
        rng = np.random.default_rng(seed)
        self.A, self.ctx = A, ctx
        self.x, self.r = (rng.standard_normal((rows, dim)).astype(np.float16) for _ in range(2))
        self.norm = (1 + 0.1 * rng.standard_normal((1, dim))).astype(np.float16)
        self.gu, self.down = ((rng.standard_normal(s) * 0.03).astype(np.float16) for s in ((2 * ffn, dim), (dim, ffn)))
        self.tx, self.tr, self.tn = (ctx.from_numpy(a) for a in (self.x, self.r, self.norm))
        self.w = []
        for m in (self.gu, self.down):
            self.w.append(A.FP8Tensor.empty(ctx, *m.shape, 128))
            A.quantize_fp8(ctx, ctx.from_numpy(m), self.w[-1])
        self.h, self.act = A.FP8Tensor.empty(ctx, rows, dim), A.FP8Tensor.empty(ctx, rows, ffn)
        self.total, self.out, self.both = ctx.tensor(rows, dim), ctx.tensor(rows, dim), ctx.tensor(rows, 2 * ffn)
        self.gate, self.up = (A.Tensor(ctx, self.both.ptr + 2 * i * ffn, rows, 2 * ffn) for i in (0, 1))

    def run(self):
        A, ctx = self.A, self.ctx
        A.rmsnorm_fp8(ctx, self.tx, self.tn, self.h, 1e-5, self.tr, self.total)
        A.gemm_fp8(ctx, self.h, self.w[0], self.both)
        A.swiglu_fp8(ctx, self.gate, self.up, self.act)
        A.gemm_fp8(ctx, self.act, self.w[1], self.out)
        A.residual_add(ctx, self.out, self.total)


@pytest.mark.parametrize("rows,dim,ffn", [(1, 256, 688), (5, 2048, 5632), (77, 288, 768), (300, 512, 1376)])
def test_mlp(A, ctx, rows, dim, ffn):
    m = Mlp(A, ctx, rows, dim, ffn, rows)
    m.run()
    h, codes, scales = norm64(m.x, m.r, m.norm, 1e-5)
    check(m.h, codes, scales, norm_eps(dim))
    w = [quantize(a.astype(np.float64), 128) for a in (m.gu, m.down)]
    for t, want in zip(m.w, w):
        check(t, *want, 2.0**-24)
    w = [(t.codes(), t.scales()) for t in m.w]
    both = m.both.numpy()
    assert_near(both, (m.h.codes(), m.h.scales()), w[0], False)
    check(m.act, *swiglu64(both[:, :ffn], both[:, ffn:]), SWIGLU_EPS)
    got = m.out.numpy().astype(np.float64) - h
    want = values(m.act.codes(), m.act.scales()) @ values(*w[1], 128).T
    # the product's rounding to f16 and the sum's, and f32's along k
    assert np.all(np.abs(got - want) <= (np.abs(want) + np.abs(want + h)) * 2.0**-11 + 1e-3 * np.abs(want).max())


def test_mlp_captured(A, ctx):
    """The calls captured on the context's stream replay as eager ones, with eager work of other sizes between."""
    hip = C.CDLL("libamdhip64.so")
    m, other = Mlp(A, ctx, 9, 512, 1376, 1), Mlp(A, ctx, 140, 512, 1376, 2)
    m.run()
    want = m.out.numpy()
    stream = C.c_void_p(A._L.aesir_ctx_stream(ctx.h))
    graph, exe = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 1) == 0
    m.run()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
    try:
        for _ in range(4):
            m.out.upload(np.full(want.shape, np.nan, np.float16))
            m.both.upload(np.full(m.both.numpy().shape, np.nan, np.float16))
            other.run()
            assert hip.hipGraphLaunch(exe, stream) == 0
            ctx.synchronize()
            assert np.array_equal(m.out.numpy().view(np.uint16), want.view(np.uint16))
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)
