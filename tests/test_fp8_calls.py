"""What the 8-bit floating-point entry points refuse, and that a refused call launches nothing: run in a child process over a
stand-in for the HIP runtime (fake_hip.cpp), so without a GPU; and the Python side's own checks."""
import os
import subprocess
import sys

import numpy as np
import pytest

from fp8_tools import NUMBERS, nearest, quantize, values

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.join(os.path.dirname(HERE), "runeforgeai-project-aesir_amd")

START = f"""
import ctypes as C, sys
F = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
sys.path.insert(0, {PKG!r})
import numpy as np
import aesir_hip as A

ctx = A.Context(64 << 20)
x, r, s, w = ctx.tensor(4, 512), ctx.tensor(4, 512), ctx.tensor(4, 512), ctx.tensor(1, 300)
q = A.FP8Tensor.empty(ctx, 4, 300)
b = A.FP8Tensor.empty(ctx, 200, 300, 128)
c = ctx.tensor(4, 200)
before = F.fake_launches()

def T(t, rows=None, cols=None, shift=0):
    return A.Tensor(ctx, t.ptr + shift if t.ptr else 0, t.rows if rows is None else rows, t.cols if cols is None else cols, t.dtype)

def Q(t, rows=None, cols=None, shift=0, scales=None):
    return A.FP8Tensor(ctx, t.ptr + shift if shift >= 0 else 0, t.scales_ptr if scales is None else scales,
                       t.rows if rows is None else rows, t.cols if cols is None else cols, t.block_rows)

def refused(code, words, call, *args):
    try:
        call(ctx, *args)
    except A.AesirError as e:
        assert e.code == code and words in str(e), (e.code, str(e))
        assert F.fake_launches() == before
        return
    assert 0, (call.__name__, words)

null = T(x)
null.ptr = None
"""


@pytest.fixture(scope="module")
def child(tmp_path_factory):
    lib = str(tmp_path_factory.mktemp("fake") / "fake_hip.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-w", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", os.path.join(HERE, "fake_hip.cpp"), "-o", lib],
                   check=True)

    def run(script):
        r = subprocess.run([sys.executable, "-c", START + script, lib], capture_output=True, text=True, timeout=100)
        assert r.returncode == 0, r.stdout + r.stderr

    return run


CODES = """
for call, args in ((A.quantize_fp8, (x,)), (A.swiglu_fp8, (x, r)), (A.rmsnorm_fp8, (x, w))):
    n = call.__name__
    refused(-1, n + ": matrix dimensions must be positive", call, *args, Q(q, rows=0))
    refused(-1, n + ": matrix dimensions must be positive", call, *args, Q(q, cols=-1))
    refused(-1, n + ": null tensor pointer", call, *args, Q(q, shift=-1))
    refused(-1, n + ": null tensor pointer", call, *args, Q(q, scales=0))
    refused(-1, n + ": codes must be 16-byte", call, *args, Q(q, shift=8))
    refused(-1, n + ": codes must be 16-byte", call, *args, Q(q, scales=q.scales_ptr + 2))
    refused(-7, n + ": more than 2^22 columns", call, *args, Q(q, cols=(1 << 22) + 1))
    refused(-7, n + ": more than 2^40 rows", call, *args, Q(q, rows=(1 << 40) + 1))
    refused(-2, n + ": tensor shape mismatch", call, *args, Q(q, rows=5))
    refused(-2, n + ": tensor shape mismatch", call, *args, Q(q, cols=513))
    for i in range(len(args) if n == "swiglu_fp8" else 1):
        def other(t):
            return (*args[:i], t, *args[i + 1:], q)
        refused(-1, n + ": tensor dimensions must be positive", call, *other(T(x, rows=0)))
        refused(-1, n + ": tensor dimensions must be positive", call, *other(T(x, cols=0)))
        refused(-2, n + ": tensor shape mismatch", call, *other(T(x, rows=3)))
        refused(-2, n + ": tensor shape mismatch", call, *other(T(x, cols=299)))
        refused(-1, n + ": null tensor pointer", call, *other(null))
        refused(-1, n + ": f16 tensors must be 2-byte aligned", call, *other(T(x, shift=1)))
        refused(-7, n + ": tensor too large", call, *other(T(x, cols=1 << 61)))
"""

NORM = """
n = "rmsnorm_fp8"
refused(-2, n + ": weight dimension mismatch", A.rmsnorm_fp8, x, T(w, cols=299), q)
refused(-1, n + ": null tensor pointer", A.rmsnorm_fp8, x, A.Tensor(ctx, None, 1, 300), q)
refused(-1, n + ": f16 tensors must be 2-byte aligned", A.rmsnorm_fp8, x, T(w, shift=1), q)
for eps in (0.0, -1e-5, float("nan")):
    refused(-1, n + ": epsilon must be positive", A.rmsnorm_fp8, x, w, q, eps)
refused(-1, n + ": a residual and the place of its sum come together", A.rmsnorm_fp8, x, w, q, 1e-5, None, s)
refused(-1, n + ": a residual and the place of its sum come together", A.rmsnorm_fp8, x, w, q, 1e-5, r, null)
for i in (0, 1):
    for t, code, words in ((T(x, rows=3), -2, "tensor shape mismatch"), (T(x, cols=200), -2, "tensor shape mismatch"),
                           (T(x, shift=1), -1, "f16 tensors must be 2-byte aligned"), (T(x, rows=0), -1, "tensor dimensions")):
        refused(code, n + ": " + words, A.rmsnorm_fp8, T(s), w, q, 1e-5, *((t, s) if i == 0 else (r, t)))
refused(-2, n + ": a sum in place has its tensor's rows", A.rmsnorm_fp8, x, w, q, 1e-5, r, T(x, cols=500))
refused(-2, n + ": a sum in place has its tensor's rows", A.rmsnorm_fp8, x, w, q, 1e-5, r, T(r, cols=500))
refused(-2, n + ": activations have blocks of one row", A.rmsnorm_fp8, T(x, rows=200, cols=300), w, b)
refused(-2, "swiglu_fp8: activations have blocks of one row", A.swiglu_fp8, T(x, rows=200, cols=300), T(x, rows=200, cols=300), b)
assert A._L.aesir_quantize_fp8(ctx.h, x.ptr, 4, 512, q.ptr, q.scales_ptr, 4, 300, 64) == -1
assert "blocks have 1 or 128 rows" in A.last_error() and F.fake_launches() == before
"""

PRODUCT = """
n, g = "gemm_fp8", A.gemm_fp8
for i, m in ((0, q), (1, b)):
    def other(t):
        return (t, b, c) if i == 0 else (q, t, c)
    refused(-1, n + ": matrix dimensions must be positive", g, *other(Q(m, rows=0)))
    refused(-1, n + ": matrix dimensions must be positive", g, *other(Q(m, cols=0)))
    refused(-1, n + ": null tensor pointer", g, *other(Q(m, shift=-1)))
    refused(-1, n + ": null tensor pointer", g, *other(Q(m, scales=0)))
    refused(-1, n + ": codes must be 16-byte", g, *other(Q(m, shift=4)))
    refused(-2, n + ": inner matrix dimension mismatch", g, *other(Q(m, cols=299)))
    refused(-7, n + ": more than 2^22 columns", g, *other(Q(m, cols=1 << 23)))
    refused(-2, n + ": output matrix shape mismatch", g, *other(Q(m, rows=m.rows + 1)))
refused(-2, n + ": output matrix shape mismatch", g, q, b, T(c, rows=5))
refused(-2, n + ": output matrix shape mismatch", g, q, b, T(c, cols=199))
refused(-1, n + ": null tensor pointer", g, q, b, A.Tensor(ctx, None, 4, 200))
refused(-1, n + ": output is not aligned to its type", g, q, b, T(c, shift=1))
refused(-1, n + ": output is not aligned to its type", g, q, b, A.Tensor(ctx, c.ptr + 2, 4, 200, np.float32))
refused(-7, n + ": output type must be F16 or F32", g, q, b, A.Tensor(ctx, c.ptr, 4, 200, np.float64))
refused(-7, n + ": output too large", g, q, b, T(c, cols=1 << 61))
for m in (4, 30, 64):
    refused(-7, n + ": output larger than one launch takes", g, Q(q, rows=m), Q(b, rows=1 << 28), T(c, rows=m, cols=1 << 28))
for t in (c, A.Tensor(ctx, c.ptr, 4, 200, np.float32)):
    refused(-7, n + ": output larger than one launch takes", g, Q(q, rows=1 << 36), b, T(t, rows=1 << 36))
refused(-7, "quantize_fp8: more elements than one launch takes", A.quantize_fp8, T(x, rows=1 << 36), Q(b, rows=1 << 36))
refused(-2, n + ": activations have blocks of one row", g, b, b, T(c, rows=200))
refused(-2, n + ": weights have blocks of 128 rows", g, q, q, T(c, cols=4))
"""

TYPES = """
f = A.Tensor(ctx, x.ptr, 4, 512, np.uint8)
refused(-7, "quantize_fp8: tensors must be f16", A.quantize_fp8, f, q)
for args in ((f, x), (x, f)):
    refused(-7, "swiglu_fp8: tensors must be f16", A.swiglu_fp8, *args, q)
    refused(-7, "rmsnorm_fp8: tensors must be f16", A.rmsnorm_fp8, *args, q)
    refused(-7, "rmsnorm_fp8: tensors must be f16", A.rmsnorm_fp8, x, w, q, 1e-5, *args)
"""


@pytest.mark.parametrize("script", [CODES, NORM, PRODUCT, TYPES])
def test_refusals(child, script):
    child(script)


def test_a_closed_context_and_a_failing_launch(child):
    child("""
for call, args in ((A.quantize_fp8, (x, q)), (A.swiglu_fp8, (x, r, q)), (A.rmsnorm_fp8, (x, w, q)), (A.gemm_fp8, (q, b, c))):
    F.fake_fail_launch(1)
    try:
        call(ctx, *args)
        assert 0, call.__name__
    except A.AesirError as e:
        assert e.code == -4 and "launch of" in str(e), str(e)
    call(ctx, *args)
    try:
        call(type("closed", (), {"h": None}), *args)
        assert 0, call.__name__
    except A.AesirError as e:
        assert e.code == -1 and "null context" in str(e)
""")


def test_fp8_tensor_shapes():
    import aesir_hip as A

    t = A.FP8Tensor(None, 0, 0, 5, 129)
    assert t.ld == 256 and t.scales_shape == (2, 5)
    assert A.FP8Tensor(None, 0, 0, 129, 1, 128).scales_shape == (2, 1)
    with pytest.raises(ValueError):
        A.FP8Tensor(None, 0, 0, 5, 129, 64)


def test_the_model_of_the_format():
    """Every code's number is its own nearest; the middle of two goes to the even one; scales bring 448 back to the largest."""
    codes = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    assert np.array_equal(nearest(NUMBERS[codes]), codes)
    lower = np.arange(126)
    assert np.array_equal(nearest((NUMBERS[lower] + NUMBERS[lower + 1]) / 2), lower + lower % 2)
    x = np.random.default_rng(0).standard_normal((130, 300))
    for tall in (1, 128):
        v = values(*quantize(x, tall), tall)
        assert np.abs(v[:, :300] - x).max() <= np.abs(x).max() * 2.0**-4 and np.all(v[:, 300:] == 0)
        assert np.isclose(np.abs(v).max(), np.abs(x).max(), rtol=1e-15)
