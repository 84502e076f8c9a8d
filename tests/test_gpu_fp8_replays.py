"""8-bit floating-point products that are cut along k, whose stretches' sums go through the context's scratch: captured into two
graphs, replayed for other inputs, with eager users of the scratch between."""
import contextlib
import ctypes as C

import numpy as np
import pytest

from fp8_routes import PRODUCTS
from test_gpu_fp8 import A, ctx, matrix, random_matrix, well  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu

SPLIT = [p[:4] for p in PRODUCTS if p[5] > 1]


class Product:
    """A product with room for its operands; inputs of a seed."""

    def __init__(self, A, ctx, M, N, K, f32):  # noqa: F811
        self.A, self.ctx, self.K, self.f32 = A, ctx, K, f32
        self.a, self.b = A.FP8Tensor.empty(ctx, M, K), A.FP8Tensor.empty(ctx, N, K, 128)
        self.c = ctx.tensor(M, N, np.float32 if f32 else np.float16)

    def load(self, seed):
        rng = np.random.default_rng(seed)
        codes, scales = random_matrix(rng, self.a.rows, self.K, 1)
        self.a.upload(codes, scales if self.f32 else scales * np.float32(2.0**-6))
        self.b.upload(*random_matrix(rng, self.b.rows, self.K, 128))

    def run(self):
        self.A.gemm_fp8(self.ctx, self.a, self.b, self.c)

    def eager(self, seed):
        self.load(seed)
        self.run()
        return self.c.numpy().view(np.uint8)


@contextlib.contextmanager
def captured(A, ctx, calls):  # noqa: F811
    """A graph of the calls; a function that launches it."""
    hip = C.CDLL("libamdhip64.so")
    stream, graph, exe = C.c_void_p(A._L.aesir_ctx_stream(ctx.h)), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 1) == 0
    for call in calls:
        call()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0

    def launch():
        assert hip.hipGraphLaunch(exe, stream) == 0

    try:
        yield launch
    finally:
        ctx.synchronize()
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


@pytest.mark.parametrize("f32", [False, True])
def test_replays_among_eager_calls(A, ctx, f32):  # noqa: F811
    sizes = [(70, 389, 2100, f32), (50, 1001, 12400, f32), (129, 3001, 8200, f32), (65, 2100, 8200, False)]
    assert set(sizes) <= set(SPLIT)
    first, second, third, other = (Product(A, ctx, *size) for size in sizes)
    want = {p: [p.eager(seed) for seed in range(3)] for p in (first, second, third)}
    want_other = other.eager(7)
    S, hd, nq, nkv = 8000, 64, 8, 2  # attention of one row whose keys are cut, which leaves its partials in the scratch
    rng = np.random.default_rng(5)
    q, k, v = (ctx.from_numpy(rng.standard_normal(s)) for s in ((1, nq * hd), (S, nkv * hd), (S, nkv * hd)))
    out = ctx.tensor(1, nq * hd)
    A.flash_attention_gqa(ctx, q, k, v, out, S, hd, nq, nkv)
    want_out = out.numpy().view(np.uint16)
    with captured(A, ctx, [first.run, second.run]) as one, captured(A, ctx, [third.run]) as two:
        for i in range(6):
            for p in (first, second, third):
                p.load(i % 3)
                p.c.upload(np.full((p.c.rows, p.c.cols), np.nan))
            other.run()
            one()
            A.flash_attention_gqa(ctx, q, k, v, out, S, hd, nq, nkv)
            two()
            other.run()
            ctx.synchronize()
            for p in (first, second, third):
                assert np.array_equal(p.c.numpy().view(np.uint8), want[p][i % 3]), i
            assert np.array_equal(out.numpy().view(np.uint16), want_out), i
            assert np.array_equal(other.c.numpy().view(np.uint8), want_other), i


@pytest.mark.parametrize("M,N,K,f32", SPLIT)
def test_same_bits_among_others(A, ctx, M, N, K, f32):  # noqa: F811
    """A product between products that leave other sums in the scratch."""
    p, q = Product(A, ctx, M, N, K, f32), Product(A, ctx, 99, 128, 4200, not f32)
    q.load(2)
    want = p.eager(1)
    for _ in range(5):
        p.c.upload(np.full((M, N), np.nan))
        for _ in range(3):
            q.run()
            p.run()
        assert np.array_equal(p.c.numpy().view(np.uint8), want)
