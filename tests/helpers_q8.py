"""Plain 64-bit forms of the 8-bit floating point operators, and the bounds
their tests use.

e4m3: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7f and 0xff are NaN,
there is no infinity, the largest value is 448 and the smallest step 2^-9.
"""
import numpy as np

from hip_backend import BF16, F16, F32, Tensor
from hip_backend.synth import f32_to_bf16_bits

U = 2.0 ** -24  # half a step of F32, relative


def _table():
    v = np.empty(256, np.float64)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[c] = -x if c & 128 else x
    v[0x7F] = v[0xFF] = np.nan
    return v


TABLE = _table()
POS = TABLE[:127]  # 0 .. 448, ascending


def decode(codes):
    return TABLE[np.asarray(codes, np.uint8)]


def encode(x):
    """Nearest e4m3 code, ties to even; beyond 464 and NaN: NaN."""
    x = np.asarray(x, np.float64)
    a = np.abs(x)
    hi = np.clip(np.searchsorted(POS, a), 1, 126)
    lo = hi - 1
    mid = (POS[lo] + POS[hi]) / 2
    c = np.where((a > mid) | ((a == mid) & (hi % 2 == 0)), hi, lo)
    c = np.where(~(a <= 464), 0x7F, c)
    return (c | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def bf16(bits):
    return (np.asarray(bits, np.uint32) << 16).view(np.float32)


def nblocks(n):
    return -(-n // 128)


def spread(s, n, axis=-1):
    return np.take(s, np.arange(n) // 128, axis=axis)


def quantize_rows(y):
    """(codes, scale bits) of rows y [rows, n] by the definition, in F32."""
    y = np.asarray(y, np.float32)
    rows, n = y.shape
    top = np.stack([np.abs(y[:, i:i + 128]).max(1) for i in range(0, n, 128)], 1)
    with np.errstate(invalid="ignore", over="ignore"):
        s = top / np.float32(448)
    s = np.where(s < np.float32(2.0 ** -126), np.float32(2.0 ** -126), s).astype(np.float32)
    bits = f32_to_bf16_bits(s).reshape(s.shape)
    with np.errstate(invalid="ignore", divide="ignore"):
        return encode(y.astype(np.float64) / spread(bf16(bits).astype(np.float64), n)), bits


def rows_value(codes, bits):
    with np.errstate(invalid="ignore"):
        return decode(codes) * spread(bf16(bits).astype(np.float64), codes.shape[1])


def random_rows(rng, rows, n, std=1.0):
    """Codes and scales of random rows."""
    return quantize_rows(rng.standard_normal((rows, n)) * std * np.exp(0.5 * rng.standard_normal(n)))


class Weight8:
    """Random e4m3 weights [E, out, in] with block scales."""

    def __init__(self, rng, E, out, n_in, scale_type=F32):
        self.shape = (E, out, n_in)
        c = rng.integers(0, 256, self.shape, dtype=np.uint8)
        c[(c & 0x7F) == 0x7F] = 0x30
        self.codes = c
        s = (2e-4 * np.exp(rng.standard_normal((E, nblocks(out), nblocks(n_in))))).astype(np.float32)
        if scale_type == F32:
            self.bits, self.scales = s, s.astype(np.float64)
        elif scale_type == BF16:
            self.bits = f32_to_bf16_bits(s).reshape(s.shape)
            self.scales = bf16(self.bits).astype(np.float64)
        else:
            assert scale_type == F16
            self.bits = s.astype(np.float16).view(np.uint16)
            self.scales = self.bits.view(np.float16).astype(np.float64)
        self.scale_type = scale_type

    def tensor(self, dense=False):
        E, out, n_in = self.shape
        dims = [n_in, out] if dense else [n_in, out, E]
        return Tensor.block8(dims, self.codes, self.bits, self.scale_type)

    def value(self, e=0):
        _, out, n_in = self.shape
        return decode(self.codes[e]) * spread(spread(self.scales[e], out, 0), n_in, 1)


def product(x, w):
    """x [T, in] . w[out, in] in 64 bits, and two magnitudes for the bounds:
    the sum of |products|, and the sum over groups of eight neighbouring columns
    of the largest |product|."""
    y = x @ w.T
    mag = np.abs(x) @ np.abs(w).T
    g = np.zeros_like(mag)
    a, b = np.abs(x), np.abs(w)
    for i in range(0, x.shape[1], 8):
        top = np.zeros_like(mag)
        for k in range(i, min(i + 8, x.shape[1])):
            np.maximum(top, a[:, k:k + 1] * b[None, :, k], out=top)
        g += top
    return y, mag, g


def f32_bound(n_in, mag):
    """F32 outputs: products are exact; 128 additions of a block, each a rounding
    of a partial sum of at most `mag`, the product of its two scales, and one
    rounding per block as it joins the running sum."""
    return (128 + 2 + nblocks(n_in)) * U * mag


def cut_bound(n_in, mag, groups):
    """Sums of the 8-bit matrix instructions: the F32 ones, and seven of eight
    products cut at 2^-13 of the largest."""
    return f32_bound(n_in, mag) + 7 * 2.0 ** -13 * groups


def silu(g):
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g))


def check_quantized(codes, bits, y, dy, cols=None):
    """Rows in 8 bits against their 64-bit values y, known to dy: a scale within
    half a bf16 step (2^-8) of max|y| / 448, a code within half a step of e4m3
    (2^-4 of the value, or half of the smallest step) of y."""
    n = y.shape[1]
    top = np.stack([np.abs(y[:, i:i + 128]).max(1) for i in range(0, n, 128)], 1)
    dtop = np.stack([dy[:, i:i + 128].max(1) for i in range(0, n, 128)], 1)
    s = bf16(bits).astype(np.float64)
    want = np.maximum(top / 448, 2.0 ** -126)
    assert np.all(np.abs(s - want) <= 2.0 ** -8 * (want + dtop / 448) + dtop / 448)
    step = spread(s, n)
    got = rows_value(codes, bits)
    lim = np.maximum(2.0 ** -4 * (np.abs(y) + dy), 2.0 ** -10 * step) + dy + 2.0 ** -20 * np.abs(y)
    bad = np.abs(got - y) > lim
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist())
