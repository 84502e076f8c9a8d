"""The 8-bit floating-point format in numpy, from its definition: e4m3 numbers, and the codes and scales of values."""
import numpy as np


def numbers():
    """The value of each of the 256 codes (NaN for 0x7f and 0xff)."""
    out = np.empty(256)
    for c in range(256):
        e, f = c >> 3 & 15, c & 7
        out[c] = (-1) ** (c >> 7) * (f / 8 * 2.0**-6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7))
    out[[127, 255]] = np.nan
    return out


NUMBERS = numbers()


def nearest(t):
    """Codes of the e4m3 numbers nearest t (float64, at most 448), ties to the even code; the sign is kept."""
    half = NUMBERS[:127]
    middle = (half[1:] + half[:-1]) / 2
    a = np.abs(t)
    i = np.searchsorted(middle, a)
    tie = (i < 126) & (middle[np.minimum(i, 125)] == a)
    return (i + (tie & (i % 2 == 1)) + 128 * np.signbit(t)).astype(np.uint8)


def quantize(y, tall=1, least=0.0):
    """Codes [rows, ld] and scales (float64; [ld / 128, rows], or [row blocks, ld / 128] where tall is 128) of the
    float64 values y. Blocks without a value of `least` are zeros."""
    rows, cols = y.shape
    nb = -(-cols // 128)
    codes = np.zeros((rows, nb * 128), np.uint8)
    scales = np.empty((-(-rows // tall), nb))
    with np.errstate(all="ignore"):
        for r in range(0, rows, tall):
            for b in range(nb):
                v = y[r:r + tall, 128 * b:128 * b + 128]
                a = np.abs(v).max()
                to = codes[r:r + tall, 128 * b:128 * b + 128]
                if not np.isfinite(v).all():
                    to[:] = 0x7F
                    a = np.nan
                elif a >= least and a > 0:
                    to[:, : v.shape[1]] = nearest(v * 448 / a)
                else:
                    a = 0.0
                scales[r // tall, b] = a / 448
    return codes, scales.T.copy() if tall == 1 else scales


def values(codes, scales, tall=1):
    """float64 values [rows, ld] of codes and scales."""
    s = scales.T if tall == 1 else np.repeat(scales, 128, 0)[: len(codes)]
    return NUMBERS[codes] * np.repeat(s.astype(np.float64), 128, 1)


def same_codes(got, want):
    """Whether codes stand for the same numbers (zeros of either sign, any NaN)."""
    return np.array_equal(NUMBERS[got], NUMBERS[want], equal_nan=True)
