"""Every kernel of the 8-bit floating-point products, and the norm's, against 64 bits: the sizes of fp8_routes.py, of which
test_fp8_routes.py shows which kernel each takes."""
import numpy as np
import pytest

from fp8_routes import NORMS, PRODUCTS
from fp8_tools import nearest, values
from test_gpu_fp8 import A, activations, check, ctx, dirty, norm64, norm_eps, product, put, random_matrix, well  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu

SIZES = [p[:4] for p in PRODUCTS]


@pytest.mark.parametrize("M,N,K,f32", SIZES)
def test_whole_numbers(A, ctx, M, N, K, f32):  # noqa: F811
    """Small whole numbers and scales that are powers of two: every sum is exact, on either matrix instruction, and f16
    results are rounded once."""
    rng = np.random.default_rng(M + N + K)
    ones = nearest(np.arange(-2.0, 3.0))
    a, b = random_matrix(rng, M, K, 1), random_matrix(rng, N, K, 128)
    for codes, scales in (a, b):
        codes[:, :K] = ones[rng.integers(0, 5, (len(codes), K))]
        scales[:] = np.exp2(rng.integers(-1, 2, scales.shape))
    want = values(*a).astype(np.float32) @ values(*b, 128).astype(np.float32).T  # every sum of these is an f32 too
    assert np.array_equal(product(A, ctx, a, b, K, f32, 3), want.astype(np.float32 if f32 else np.float16))


def bound(x, w, f32, want):
    """Additions along k a unit of f32's last place each, a block's scales and their products half a one each; for f16 what the
    8-bit matrix instruction drops of 8 neighbouring products, 2^-13 of the largest each (the largest is at most the
    product of the largest factors), and half a step of f16 or of its least number."""
    b = np.abs(x) @ np.abs(w).T * ((x.shape[1] + 8) * 2.0**-23)
    if not f32:
        top = [np.abs(v).reshape(len(v), -1, 8).max(2) for v in (x, w)]
        b += top[0] @ top[1].T * (8 * 2.0**-13)
        b += np.abs(want) * 2.0**-11 + 2.0**-25
    return b


@pytest.mark.parametrize("M,N,K,f32", SIZES)
def test_roundings_and_nan(A, ctx, M, N, K, f32):  # noqa: F811
    """Codes of all numbers; the same bits a second time; then NaN codes and scales, which reach their rows of A and of B only."""
    rng = np.random.default_rng(M * 7 + N * 3 + K)
    a, b = random_matrix(rng, M, K, 1), random_matrix(rng, N, K, 128)
    if not f32:
        a = (a[0], a[1] * 2.0**-6)  # within f16
    x, w = values(*a), values(*b, 128)
    want = x @ w.T
    got = product(A, ctx, a, b, K, f32)
    off = np.abs(got.astype(np.float64) - want)
    b_ = bound(x, w, f32, want)
    assert np.all(off <= b_), (np.argwhere(~(off <= b_))[:4], np.max(off / b_))
    assert np.array_equal(product(A, ctx, a, b, K, f32, 1).view(np.uint8), got.view(np.uint8))

    nan = np.zeros((M, N), bool)
    a[0][M // 2, K - 1], b[0][N // 3, K // 2], b[0][N - 1, 0] = 0x7F, 0xFF, 0x7F
    nan[M // 2], nan[:, [N // 3, N - 1]] = True, True
    if N > 256:
        b[1][1, 2] = np.nan
        nan[:, 128:256] = True
    if M > 4:
        a[1][1, M - 2] = np.nan
        nan[M - 2] = True
    with_nan = product(A, ctx, a, b, K, f32)
    assert np.array_equal(np.isnan(with_nan), nan)
    assert np.array_equal(with_nan[~nan], got[~nan])


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("cols", [cols for cols, _ in NORMS])
def test_norm(A, ctx, cols, residual):  # noqa: F811
    """On each width; with a row that holds a NaN, one of zeros, and the sum in place of x."""
    rng = np.random.default_rng(cols)
    x, r = activations(rng, 7, cols), activations(rng, 7, cols)
    w = (1 + 0.3 * rng.standard_normal((1, cols))).astype(np.float16)
    x[5, cols - 1] = np.nan
    x[6], r[6] = 0, 0
    t, tx = dirty(A, ctx, 7, cols), put(A, ctx, x)
    h, codes, scales = norm64(x, r if residual else None, w, 1e-5)
    A.rmsnorm_fp8(ctx, tx, put(A, ctx, w), t, 1e-5, *((put(A, ctx, r), tx) if residual else ()))
    assert np.array_equal(tx.numpy(), h, equal_nan=True)
    check(t, codes, scales, norm_eps(cols))
