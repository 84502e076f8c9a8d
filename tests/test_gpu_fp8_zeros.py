"""Blocks that are zeros in 8-bit floating point: scale 0 and code bytes 0, whatever the signs of the values they come from."""
import numpy as np
import pytest

from fp8_tools import same_codes
from test_gpu_fp8 import A, ctx, dirty, norm64, put, swiglu64, well  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu


def assert_zeros(t, blocks):
    """blocks: (row, column block) of those that are zeros."""
    codes, scales = t.codes(), t.scales()
    for r, b in blocks:
        assert np.all(codes[r, 128 * b:128 * b + 128] == 0), (r, b, np.unique(codes[r, 128 * b:128 * b + 128]))
        at = scales[b, r] if t.block_rows == 1 else scales[r // 128, b]
        assert at.view(np.uint32) == 0, (r, b, at)


@pytest.mark.parametrize("cols", [128, 200, 2056])
def test_quantize_negative_zeros(A, ctx, cols):  # noqa: F811
    x = np.random.default_rng(cols).standard_normal((140, cols)).astype(np.float16)
    x[3], x[5, :128] = -0.0, np.where(np.arange(128) % 2, -0.0, 0.0)
    t = dirty(A, ctx, 140, cols)
    A.quantize_fp8(ctx, put(A, ctx, x), t)
    assert_zeros(t, [(3, b) for b in range(-(-cols // 128))] + [(5, 0)])


def test_quantize_weights_negative_zeros(A, ctx):  # noqa: F811
    x = np.random.default_rng(1).standard_normal((200, 300)).astype(np.float16)
    x[:128, 128:256] = -0.0
    t = dirty(A, ctx, 200, 300, 128)
    A.quantize_fp8(ctx, put(A, ctx, x), t)
    assert_zeros(t, [(r, 1) for r in range(128)])


@pytest.mark.parametrize("cols", [300, 4096, 5000, 20000])
def test_norm_negative_zeros(A, ctx, cols):  # noqa: F811
    """-0 rows, sums that are -0, and negative values times a weight of 0."""
    rng = np.random.default_rng(cols)
    x, r = rng.standard_normal((2, 4, cols)).astype(np.float16)
    w = rng.standard_normal((1, cols)).astype(np.float16)
    x[1], r[1] = -0.0, -0.0
    w[0, 128:256] = 0
    x[:, 128:256] = -np.abs(x[:, 128:256])
    for residual in (None, r):
        t = dirty(A, ctx, 4, cols)
        more = () if residual is None else (put(A, ctx, residual), put(A, ctx, np.zeros_like(x)))
        A.rmsnorm_fp8(ctx, put(A, ctx, x), put(A, ctx, w), t, 1e-5, *more)
        assert_zeros(t, [(1, b) for b in range(-(-cols // 128))] + [(i, 1) for i in range(4)])
        assert same_codes(t.codes(), norm64(x, residual, w, 1e-5)[1])


def test_swiglu_negative_zeros(A, ctx):  # noqa: F811
    """Values of -0 and negative ones under 2^-64, in blocks that f32 decides and in blocks next to the border, which f64 does."""
    rng = np.random.default_rng(2)
    g, u = rng.standard_normal((2, 6, 384)).astype(np.float16)
    g[1], u[2] = -0.0, -0.0
    g[3], u[3] = -60, 1  # y about -5e-25
    g[4], u[4] = np.where(np.arange(384) % 2, -70, 0), 2
    t = dirty(A, ctx, 6, 384)
    A.swiglu_fp8(ctx, put(A, ctx, g), put(A, ctx, u), t)
    assert_zeros(t, [(r, b) for r in (1, 2, 3, 4) for b in range(3)])
    g = np.linspace(-50, -44, 128 * 64).astype(np.float16).reshape(64, 128)
    t = dirty(A, ctx, 64, 128)
    A.swiglu_fp8(ctx, put(A, ctx, g), put(A, ctx, np.full_like(g, 0.75)), t)
    scales = swiglu64(g, np.full_like(g, 0.75))[1]
    assert (scales == 0).any() and (scales > 0).any()
    assert_zeros(t, [(r, 0) for r in np.flatnonzero(scales[0] == 0)])
