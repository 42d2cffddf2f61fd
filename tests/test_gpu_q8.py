"""The 8-bit floating point operators on the GPU, through the public entry
points, against their 64-bit forms (helpers_q8)."""
import numpy as np
import pytest

from helpers_q8 import (POS, U, Weight8, bf16, check_quantized, cut_bound, decode, encode, f32_bound, nblocks, product,
                        quantize_rows, random_rows, rows_value, silu, spread)
from hip_backend import BF16, E4M3, F16, F32, Batch, Buffer, Gpu, Rows8, ShapeError, Tensor
from hip_backend.api import MoeBufferC, MoeRegionC
from hip_backend.synth import f32_to_bf16_bits

pytestmark = pytest.mark.gpu


class Owned:
    """Allocations of one test, released at its end."""

    def __init__(self, gpu):
        self.gpu, self.bufs = gpu, []

    def upload(self, a):
        b = self.gpu.upload(np.asarray(a))
        self.bufs.append(b)
        return b

    def u32(self, a):
        b = self.gpu.upload_u32(np.asarray(a))
        self.bufs.append(b)
        return b

    def zeros(self, n, fill=None):
        b = self.gpu.zeros(n)
        self.bufs.append(b)
        if fill is not None:
            self.gpu.write(b, np.full(n, fill, np.uint32).view(np.float32))
        return b

    def rows8(self, rows, n, codes=None, scales=None):
        r = self.gpu.rows8(rows, n, codes, scales)
        self.bufs += r.buffers
        return r

    def weight(self, t):
        w = self.gpu.weight_tensor(t)
        self.bufs += [Buffer(self.gpu, MoeBufferC(), r.ptr) for r in w.regions]
        return w

    def release(self):
        for b in self.bufs:
            self.gpu.release(b)


@pytest.fixture
def own(gpu):
    o = Owned(gpu)
    yield o
    o.release()


def read_bf16(gpu, b):
    return bf16(gpu.read_u32(b).view(np.uint16)).astype(np.float64)


# ------------------------------------------------------------------- norm --
def norm64(x, w, eps):
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(1, keepdims=True) + eps) * w


NORM_SIZES = [(1, 16), (1, 2048), (3, 128), (2, 144), (5, 1360), (7, 2064), (2, 4096), (3, 6160), (2, 9232)]


@pytest.mark.parametrize("rows,n", NORM_SIZES)
@pytest.mark.parametrize("wtype", [F32, F16, BF16])
def test_norm_q8(gpu, own, rows, n, wtype):
    rng = np.random.default_rng(rows * 10000 + n)
    x = (rng.standard_normal((rows, n)) * 3).astype(np.float32)
    r = rng.standard_normal((rows, n)).astype(np.float32)
    w = (1 + 0.3 * rng.standard_normal(n)).astype(np.float32)
    if wtype == F16:
        raw = w.astype(np.float16)
        w64, t = raw.astype(np.float64), Tensor.dense([n], raw.view(np.uint16), F16)
    elif wtype == BF16:
        raw = f32_to_bf16_bits(w)
        w64, t = bf16(raw).astype(np.float64), Tensor.dense([n], raw, BF16)
    else:
        w64, t = w.astype(np.float64), Tensor.dense([n], w)
    wd, xb, rb = own.weight(t), own.upload(x), own.upload(r)
    for resid, with_sum, with_y in [(True, True, True), (False, False, True), (True, False, False),
                                    (False, True, False)]:
        q, s, y = own.rows8(rows, n), own.zeros(rows * n), own.zeros(rows * n)
        with gpu.batch() as b:
            b.norm_q8(xb, rb if resid else None, wd, s if with_sum else None, y if with_y else None, q, 1e-6)
        sum_ = x + r if resid else x
        if with_sum:
            assert np.array_equal(gpu.read(s).reshape(rows, n), sum_)
        want = norm64(sum_, w64, 1e-6)
        # the mean of n squares in sums of at most 64 roundings, its root and
        # reciprocal, and two products
        dy = (64 + 6) * U * np.abs(want)
        codes, bits = gpu.read_rows8(q)
        if with_y:
            got = gpu.read(y).reshape(rows, n)
            assert np.all(np.abs(got - want) <= dy)
            # the scale is that of the F32 values written beside the codes
            assert np.array_equal(bits, quantize_rows(got)[1])
        check_quantized(codes, bits, want, dy)


def test_norm_q8_in_place(gpu, own):
    rng = np.random.default_rng(5)
    rows, n = 3, 6160
    x = rng.standard_normal((rows, n)).astype(np.float32)
    r = rng.standard_normal((rows, n)).astype(np.float32)
    wd = own.weight(Tensor.dense([n], np.ones(n, np.float32)))
    out = []
    for where in ("own", "x", "residual"):
        xb, rb, q = own.upload(x), own.upload(r), own.rows8(rows, n)
        s = {"own": own.zeros(rows * n), "x": xb, "residual": rb}[where]
        with gpu.batch() as b:
            b.norm_q8(xb, rb, wd, s, None, q, 1e-5)
        assert np.array_equal(gpu.read(s).reshape(rows, n), x + r)
        out.append(gpu.read_rows8(q))
    for c, s in out[1:]:
        assert np.array_equal(c, out[0][0]) and np.array_equal(s, out[0][1])


def test_norm_q8_from_unaligned_buffers(gpu, own):
    """F32 arrays that start at any element."""
    rng = np.random.default_rng(6)
    rows, n = 2, 400
    x = rng.standard_normal(rows * n + 3).astype(np.float32)
    wd = own.weight(Tensor.dense([n], np.ones(n, np.float32)))
    xb, y, s = own.upload(x), own.zeros(rows * n + 1), own.zeros(rows * n + 2)
    q = own.rows8(rows, n)
    with gpu.batch() as b:
        b.norm_q8(xb.view(3, rows * n), None, wd, s.view(2, rows * n), y.view(1, rows * n), q, 1e-6)
    want = norm64(x[3:].reshape(rows, n), np.ones(n), 1e-6)
    assert np.all(np.abs(gpu.read(y)[1:].reshape(rows, n) - want) <= 70 * U * np.abs(want))
    assert np.array_equal(gpu.read(s)[2:], x[3:]) and gpu.read(y)[0] == 0
    check_quantized(*gpu.read_rows8(q), want, 70 * U * np.abs(want))


def test_norm_q8_of_zeros_tiny_and_non_finite_rows(gpu, own):
    rows, n = 5, 272
    rng = np.random.default_rng(7)
    x = rng.standard_normal((rows, n)).astype(np.float32)
    x[0] = 0
    x[1, :128] = 0
    w = np.ones(n, np.float32)
    w[256:] = 1e-38                     # values below 448 * 2^-126
    x[2, 3], x[3, 200] = np.inf, np.nan
    wd, xb, q = own.weight(Tensor.dense([n], w)), own.upload(x), own.rows8(rows, n)
    with gpu.batch() as b:
        b.norm_q8(xb, None, wd, None, None, q, 1e-6)
    codes, bits = gpu.read_rows8(q)
    least = f32_to_bf16_bits(np.array([2.0 ** -126], np.float32))[0]
    assert np.all(codes[0] & 0x7F == 0) and np.all(bits[0] == least)
    assert np.all(codes[1, :128] & 0x7F == 0) and bits[1, 0] == least and bits[1, 1] != least and bits[1, 2] == least
    v = rows_value(codes, bits)
    assert np.isnan(v[3]).all()                        # NaN in the sum of squares
    assert np.isnan(v[2, :128]).all()                  # inf * 0
    want = norm64(x[4:], w.astype(np.float64), 1e-6)
    check_quantized(codes[4:], bits[4:], want, 70 * U * np.abs(want) + 2.0 ** -149)


@pytest.mark.parametrize("least", [False, True])
def test_norm_q8_codes_of_quotients_between_two_codes(gpu, own, least):
    """Rows of ones and minus ones have the norm's weights as their values: those
    are each middle between two codes times each mantissa of a scale, and the
    F32 values next to it.  The codes are those of the quotient in F32."""
    mids = (POS[:-1] + POS[1:]) / 2
    scales = np.array([2.0 ** -126] if least else (1 + np.arange(128) / 128) * 2.0 ** -9)
    exact = np.zeros((len(scales), 128), np.float32)
    exact[:, 0] = 448 * scales
    exact[:, 1:127] = scales[:, None] * mids
    assert np.array_equal(exact[:, 1:127].astype(np.float64), scales[:, None] * mids)
    x = np.where(np.arange(exact.size) % 3 == 1, -1, 1).astype(np.float32)
    for w in (exact, np.nextafter(exact, np.float32(0)), np.nextafter(exact, np.float32(np.inf))):
        w = w.copy()
        w[:, 0] = exact[:, 0]
        for part in (w.ravel(), w.ravel()[:min(w.size, 2048)]):   # a long row; one that stays in registers
            n = part.size
            wd, xb, y, q = own.weight(Tensor.dense([n], part)), own.upload(x[:n]), own.zeros(n), own.rows8(1, n)
            with gpu.batch() as b:
                b.norm_q8(xb, None, wd, None, y, q, 1e-30)
            v = gpu.read(y)
            assert np.array_equal(v, x[:n] * part)
            codes, bits = gpu.read_rows8(q)
            s = spread(bf16(bits[0]), n)
            assert np.array_equal(s, spread(scales, n).astype(np.float32))
            assert np.array_equal(codes[0], encode((v / s).astype(np.float64)))


# ------------------------------------------------------------------ dense --
def check_rows(got, want, mag, groups, n_in, bf):
    if bf:
        # the output's rounding: half a bf16 step, 2^-8 of the value
        lim = cut_bound(n_in, mag, groups)
        lim = lim + 2.0 ** -8 * (np.abs(want) + lim)
    else:
        lim = f32_bound(n_in, mag)
    bad = ~(np.abs(got - want) <= lim)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(),
                           float(np.max(np.abs(got - want) / np.maximum(lim, 1e-300))))


MATMUL_SIZES = [(1, 128, 64), (1, 16, 1), (2, 48, 15), (1, 2048, 512), (15, 144, 130), (16, 256, 256), (17, 272, 258),
                (33, 640, 300), (64, 128, 1000), (100, 1040, 512), (129, 256, 64), (300, 384, 770)]


@pytest.mark.parametrize("T,n_in,out", MATMUL_SIZES)
@pytest.mark.parametrize("y_type", [F32, BF16])
def test_matmul_q8(gpu, own, T, n_in, out, y_type):
    if y_type == BF16 and T * out % 2:
        pytest.skip("bf16 outputs come two to an element")
    rng = np.random.default_rng(T * 1000 + n_in + out)
    st = [F32, BF16, F16][(T + out) % 3]
    w = Weight8(rng, 1, out, n_in, st)
    codes, bits = random_rows(rng, T, n_in)
    wd, x = own.weight(w.tensor(dense=True)), own.rows8(T, n_in, codes, bits)
    elems = T * out if y_type == F32 else T * out // 2
    y = own.zeros(elems + 4, 0x7F7F7F7F)
    with gpu.batch() as b:
        b.matmul_q8(wd, x, y.view(0, elems), y_type)
    want, mag, g = product(rows_value(codes, bits), w.value())
    got = gpu.read(y.view(0, elems)) if y_type == F32 else read_bf16(gpu, y.view(0, elems))
    check_rows(got.reshape(T, out), want, mag, g, n_in, y_type == BF16)
    assert np.all(gpu.read_u32(y)[elems:] == 0x7F7F7F7F)   # nothing past the output


@pytest.mark.parametrize("y_type", [F32, BF16])
@pytest.mark.parametrize("T", [1, 40, 200])
def test_matmul_q8_every_code(gpu, own, T, y_type):
    """One-hot rows read each code of a weight back exactly, at every column."""
    rng = np.random.default_rng(11)
    n_in, out = 256, 256
    w = Weight8(rng, 1, out, n_in)
    w.codes[0, :, :] = (np.arange(out)[:, None] + np.arange(n_in)[None, :]) % 256
    w.codes[0, 4:][(w.codes[0, 4:] & 0x7F) == 0x7F] = 0x30   # NaN in the first four rows only
    w.scales[:], w.bits[:] = 1, 1
    wd = own.weight(w.tensor(dense=True))
    cols = (np.arange(T) * 37) % n_in
    codes = np.zeros((T, n_in), np.uint8)
    codes[np.arange(T), cols] = encode(1.0)
    x = own.rows8(T, n_in, codes, np.full((T, 2), 0x3F80, np.uint16))
    y = own.zeros(T * out if y_type == F32 else T * out // 2)
    with gpu.batch() as b:
        b.matmul_q8(wd, x, y, y_type)
    got = (gpu.read(y) if y_type == F32 else read_bf16(gpu, y)).reshape(T, out)
    v = decode(w.codes[0])
    nan = np.isnan(v).any(1)            # a NaN of the row reaches every token (NaN * 0)
    assert nan.sum() == 4 and np.isnan(got[:, nan]).all()
    assert np.array_equal(got[:, ~nan], v[:, cols].T[:, ~nan])


def test_matmul_q8_wide_scales(gpu, own):
    """Scales and values over their whole range; a NaN or infinite scale."""
    rng = np.random.default_rng(12)
    T, n_in, out = 20, 512, 384
    w = Weight8(rng, 1, out, n_in)
    w.bits[:] = (2.0 ** rng.integers(-60, 20, w.bits.shape)).astype(np.float32)
    w.scales[:] = w.bits
    codes, _ = random_rows(rng, T, n_in)
    bits = f32_to_bf16_bits((2.0 ** rng.integers(-40, 40, (T, 4))).astype(np.float32)).reshape(T, 4)
    bits[3, 1], bits[4, 2] = 0x7FC0, 0x7F80
    wd, x, y = own.weight(w.tensor(dense=True)), own.rows8(T, n_in, codes, bits), own.zeros(T * out)
    with gpu.batch() as b:
        b.matmul_q8(wd, x, y)
    got = gpu.read(y).reshape(T, out).astype(np.float64)
    assert np.isnan(got[3]).all() and not np.isfinite(got[4]).any()
    keep = [t for t in range(T) if t not in (3, 4)]
    want, mag, g = product(rows_value(codes, bits)[keep], w.value())
    check_rows(got[keep], want, mag, g, n_in, False)


# ---------------------------------------------------------------- experts --
def segments(rng, lens, shuffle=True):
    """offsets and perm of segments of these lengths (pairs in a random order
    across segments, ascending within one, as a dispatch gives them)."""
    P = int(sum(lens))
    offsets = np.concatenate([[0], np.cumsum(lens)]).astype(np.uint32)
    perm = rng.permutation(P) if shuffle else np.arange(P)
    for a, b in zip(offsets[:-1], offsets[1:]):
        perm[a:b] = np.sort(perm[a:b])
    return offsets, perm.astype(np.uint32)


LENS = [
    [1], [0, 1, 0], [2, 0, 0, 16, 1, 15, 17], [33, 0, 64, 5, 1], [100, 31, 0, 129],
    [0] * 300 + [3] + [0] * 800 + [1, 2],        # more experts than threads, nearly all empty
    [260, 4], [70, 96, 65, 97],
]


@pytest.mark.parametrize("lens", LENS, ids=lambda v: f"{len(v)}x{sum(v)}")
@pytest.mark.parametrize("n_in,out", [(128, 64), (48, 300), (272, 130)])
@pytest.mark.parametrize("y_type", [F32, BF16])
def test_expert_matmul_q8(gpu, own, lens, n_in, out, y_type):
    rng = np.random.default_rng(sum(lens) + n_in)
    E, P = len(lens), sum(lens)
    w = Weight8(rng, E, out, n_in, [F32, BF16, F16][P % 3])
    codes, bits = random_rows(rng, P, n_in)
    offsets, perm = segments(rng, lens)
    wd, x = own.weight(w.tensor()), own.rows8(P, n_in, codes, bits)
    ob, pb = own.u32(offsets), own.u32(perm)
    v = rows_value(codes, bits)
    want, mag, g = (np.zeros((P, out)) for _ in range(3))
    for e in range(E):
        a, b_ = offsets[e], offsets[e + 1]
        if b_ > a:
            want[a:b_], mag[a:b_], g[a:b_] = product(v[a:b_], w.value(e))
    elems = P * out if y_type == F32 else P * out // 2
    for p in (pb, None):
        y = own.zeros(elems)
        with gpu.batch() as b:
            b.expert_matmul_q8(wd, x, ob, p, y, y_type)
        got = (gpu.read(y) if y_type == F32 else read_bf16(gpu, y)).reshape(P, out)
        if p is not None:
            got = got[perm]
        check_rows(got, want, mag, g, n_in, y_type == BF16)


def swiglu64(x, gate, up, e):
    """The SwiGLU of expert e in 64 bits and how far 8-bit sums may be off:
    |silu'| <= 1.1, and eight roundings of the exponential, division and products."""
    n_in = x.shape[1]
    g, gm, gg = product(x, gate.value(e))
    u, um, ug = product(x, up.value(e))
    dg, du = cut_bound(n_in, gm, gg), cut_bound(n_in, um, ug)
    a = silu(g) * u
    return a, 1.1 * dg * (np.abs(u) + du) + np.abs(silu(g)) * du + 8 * U * np.abs(a)


@pytest.mark.parametrize("lens", LENS, ids=lambda v: f"{len(v)}x{sum(v)}")
@pytest.mark.parametrize("n_in,ff", [(128, 64), (48, 272), (272, 16), (256, 128)])
def test_expert_swiglu_q8(gpu, own, lens, n_in, ff):
    rng = np.random.default_rng(sum(lens) * 3 + n_in)
    E, P = len(lens), sum(lens)
    st = [F32, BF16, F16][(P + ff // 16) % 3]
    gate, up = Weight8(rng, E, ff, n_in, st), Weight8(rng, E, ff, n_in, st)
    offsets, perm = segments(rng, lens)
    gd, ud, ob, pb = own.weight(gate.tensor()), own.weight(up.tensor()), own.u32(offsets), own.u32(perm)
    for K in [k for k in (1, 2, 3) if P % k == 0]:
        T = P // K
        codes, bits = random_rows(rng, T, n_in)
        x, q = own.rows8(T, n_in, codes, bits), own.rows8(P, ff)
        with gpu.batch() as b:
            b.expert_swiglu_q8(gd, ud, x, ob, pb, K, q)
        v = rows_value(codes, bits)[perm // K]
        want, dw = np.zeros((P, ff)), np.zeros((P, ff))
        for e in range(E):
            a, b_ = offsets[e], offsets[e + 1]
            if b_ > a:
                want[a:b_], dw[a:b_] = swiglu64(v[a:b_], gate, up, e)
        check_quantized(*gpu.read_rows8(q), want, dw)
    # no perm: position p reads row p
    codes, bits = random_rows(rng, P, n_in)
    x, q, q2 = own.rows8(P, n_in, codes, bits), own.rows8(P, ff), own.rows8(P, ff)
    ident = own.u32(np.arange(P))
    with gpu.batch() as b:
        b.expert_swiglu_q8(gd, ud, x, ob, None, 1, q)
        b.expert_swiglu_q8(gd, ud, x, ob, ident, 1, q2)
    for i, j in zip(gpu.read_rows8(q), gpu.read_rows8(q2)):
        assert np.array_equal(i, j)


def test_expert_products_leave_other_rows(gpu, own):
    """Positions behind the last segment, and positions whose perm names no
    row, keep what they held; ends past the positions count as their number."""
    rng = np.random.default_rng(21)
    n_in, ff, E, P = 128, 48, 3, 40
    gate, up, down = (Weight8(rng, E, ff, n_in) for _ in range(3))
    gd, ud, dd = (own.weight(w.tensor()) for w in (gate, up, down))
    codes, bits = random_rows(rng, P, n_in)
    x = own.rows8(P, n_in, codes, bits)
    perm = rng.permutation(P).astype(np.uint32)
    for offsets, live in [([0, 5, 5, 30], np.arange(30)), ([0, 7, 20, 1000], np.arange(40)),
                          ([3, 9, 2, 12], np.r_[3:9, 2:12]), ([50, 60, 70, 4000000000], np.arange(0))]:
        p2 = perm.copy()
        p2[8], p2[11] = 40, 0xFFFFFFFF
        ob, pb = own.u32(np.array(offsets, np.uint32)), own.u32(p2)
        q, y = own.rows8(P, ff, np.full((P, ff), 0x55, np.uint8), np.full((P, 1), 0x1234, np.uint16)), own.zeros(P * ff, 0x55555555)
        with gpu.batch() as b:
            b.expert_swiglu_q8(gd, ud, x, ob, pb, 1, q)
            b.expert_matmul_q8(dd, x, ob, pb, y)
        written = np.zeros(P, bool)
        written[live] = True
        written[[8, 11]] = False
        c, s = gpu.read_rows8(q)
        assert np.all(c[~written] == 0x55) and np.all(s[~written] == 0x1234)
        assert not np.any(s[written] == 0x1234)
        rows = gpu.read_u32(y).reshape(P, ff)
        to = np.zeros(P, bool)
        to[p2[written]] = True
        assert np.all(rows[~to] == 0x55555555) and not np.any((rows[to] == 0x55555555).all(1))


# Segments of enough rows for tiles of 128 (8-bit outputs; bf16 from 12, F32 from 16 a segment).
TILED = [
    [2600], [33, 0, 64, 5, 1, 2500], [100, 31, 0, 129, 2400, 0, 96, 97], [260] * 10 + [4], [128] * 21,
    [3, 0, 1, 0, 2, 43] * 17 + [500],
]


@pytest.mark.parametrize("lens", TILED, ids=lambda v: f"{len(v)}x{sum(v)}")
@pytest.mark.parametrize("n_in,out", [(128, 64), (48, 300), (272, 130), (1040, 258)])
@pytest.mark.parametrize("y_type,times", [(F32, 2), (BF16, 1)])
def test_expert_matmul_q8_of_many_rows(gpu, own, lens, n_in, out, y_type, times):
    rng = np.random.default_rng(sum(lens) + n_in)
    lens = [n * times for n in lens]
    E, P = len(lens), sum(lens)
    w = Weight8(rng, E, out, n_in, [F32, BF16, F16][P % 3])
    codes, bits = random_rows(rng, P, n_in)
    offsets, perm = segments(rng, lens)
    wd, x = own.weight(w.tensor()), own.rows8(P, n_in, codes, bits)
    ob, pb = own.u32(offsets), own.u32(perm)
    v = rows_value(codes, bits)
    elems = P * out if y_type == F32 else P * out // 2
    y = own.zeros(elems + 4, 0x7F7F7F7F)
    seen = []
    for at, p in ((0, pb), (0, None), (1, pb)):   # whole lines, no perm, rows that start unaligned
        with gpu.batch() as b:
            b.expert_matmul_q8(wd, x, ob, p, y.view(at, elems), y_type)
        g = y.view(at, elems)
        got = (gpu.read(g) if y_type == F32 else read_bf16(gpu, g)).reshape(P, out)
        seen.append(got[perm] if p is not None else got)
        assert np.all(gpu.read_u32(y)[elems + at:] == 0x7F7F7F7F)
    assert np.array_equal(seen[0], seen[1]) and np.array_equal(seen[0], seen[2])
    for e in range(E):
        a, b_ = offsets[e], offsets[e + 1]
        if b_ > a:
            check_rows(seen[0][a:b_], *product(v[a:b_], w.value(e)), n_in, y_type == BF16)


@pytest.mark.parametrize("lens", TILED, ids=lambda v: f"{len(v)}x{sum(v)}")
@pytest.mark.parametrize("n_in,ff", [(128, 64), (48, 272), (272, 16), (1040, 144)])
def test_expert_swiglu_q8_of_many_rows(gpu, own, lens, n_in, ff):
    rng = np.random.default_rng(sum(lens) * 3 + n_in)
    E, P = len(lens), sum(lens)
    K = 2 if P % 2 == 0 else 1
    st = [F32, BF16, F16][(P + ff // 16) % 3]
    gate, up = Weight8(rng, E, ff, n_in, st), Weight8(rng, E, ff, n_in, st)
    offsets, perm = segments(rng, lens)
    codes, bits = random_rows(rng, P // K, n_in)
    x, q = own.rows8(P // K, n_in, codes, bits), own.rows8(P, ff)
    gd, ud, ob, pb = own.weight(gate.tensor()), own.weight(up.tensor()), own.u32(offsets), own.u32(perm)
    with gpu.batch() as b:
        b.expert_swiglu_q8(gd, ud, x, ob, pb, K, q)
    got, gs = gpu.read_rows8(q)
    v = rows_value(codes, bits)[perm // K]
    for e in range(E):
        a, b_ = offsets[e], offsets[e + 1]
        if b_ > a:
            check_quantized(got[a:b_], gs[a:b_], *swiglu64(v[a:b_], gate, up, e))


SKIPS = [
    lambda P: ([0, P // 6, P // 6, P // 4 * 3], None),                           # positions behind the last segment
    lambda P: ([0, P // 4, P // 3 * 2, 4 * P], None),                            # an end past the positions
    lambda P: ([P // 10, P // 10 + 1, P - 1, P - 1], None),                      # before the first one
    lambda P: ([P // 4, P // 2, P // 5, P // 5 * 2], (P // 4, P // 5 * 2)),      # an end before its start, an overlap
    lambda P: ([P + 10, 2 * P, 3 * P, 4000000000], None),                        # none
]


@pytest.mark.parametrize("skip", range(len(SKIPS)))
@pytest.mark.parametrize("P,n_in,out,K", [(60, 272, 272, 2), (3000, 272, 272, 1), (3000, 128, 144, 2), (6000, 144, 130, 1)])
def test_rows_left_as_they_were_in_every_form(gpu, own, P, n_in, out, K, skip):
    """Segments that leave positions out and perms that name no row, over few rows
    and in tiles of 128: what no position names keeps what it held, the rest is
    its product."""
    rng = np.random.default_rng(P + n_in + skip)
    offsets, twice = SKIPS[skip](P)
    E = len(offsets) - 1
    gate, up, down = (Weight8(rng, E, out, n_in) for _ in range(3))
    perm = rng.permutation(P).astype(np.uint32)
    named = np.ones(P, bool)
    for i, at in enumerate((0, P // 8, P // 4, P // 3, P - 1)):
        perm[at], named[at] = (P, 0xFFFFFFFF, P + 1)[i % 3], False
    inside, expert = np.zeros(P, bool), np.zeros(P, np.int64)
    for e in range(E):
        inside[offsets[e]:offsets[e + 1]] = True
        expert[offsets[e]:offsets[e + 1]] = e
    written, sure = inside & named, inside & named
    if twice:                                   # rows of two segments: of either
        sure = sure.copy()
        sure[twice[0]:twice[1]] = False
    ob, pb = own.u32(np.array(offsets, np.uint32)), own.u32(perm)
    if out % 16 == 0:
        gd, ud = own.weight(gate.tensor()), own.weight(up.tensor())
        codes, bits = random_rows(rng, P // K, n_in)
        x = own.rows8(P // K, n_in, codes, bits)
        q = own.rows8(P, out, np.full((P, out), 0x55, np.uint8), np.full((P, nblocks(out)), 0x1234, np.uint16))
        with gpu.batch() as b:
            b.expert_swiglu_q8(gd, ud, x, ob, pb, K, q)
        c, s = gpu.read_rows8(q)
        assert np.all(c[~written] == 0x55) and np.all(s[~written] == 0x1234) and not np.any(s[written] == 0x1234)
        for e in range(E):
            at = np.flatnonzero(sure & (expert == e))
            if at.size:
                check_quantized(c[at], s[at], *swiglu64(rows_value(codes, bits)[perm[at] // K], gate, up, e))
    dd = own.weight(down.tensor())
    codes, bits = random_rows(rng, P, n_in)
    x, v = own.rows8(P, n_in, codes, bits), rows_value(codes, bits)
    to = np.zeros(P, bool)
    to[perm[written]] = True
    for y_type in (F32, BF16):
        y = own.zeros(P * out // (2 if y_type == BF16 else 1), 0x55555555)
        with gpu.batch() as b:
            b.expert_matmul_q8(dd, x, ob, pb, y, y_type)
        raw = gpu.read_u32(y).view(np.uint8).reshape(P, -1)
        assert np.all(raw[~to] == 0x55) and not np.any((raw[to] == 0x55).all(1))
        got = (gpu.read(y) if y_type == F32 else read_bf16(gpu, y)).reshape(P, out)
        for e in range(E):
            at = np.flatnonzero(sure & (expert == e))
            if at.size:
                check_rows(got[perm[at]], *product(v[at], down.value(e)), n_in, y_type == BF16)


@pytest.mark.parametrize("T,y_type", [(200, F32), (5200, F32), (200, BF16), (2600, BF16)])
@pytest.mark.parametrize("n_in", [256, 272])
def test_every_code_in_every_form(gpu, own, T, y_type, n_in):
    """As above, in tiles too and with a last block that is not whole."""
    out = 256
    w = Weight8(np.random.default_rng(11), 1, out, n_in)
    w.codes[0, :, :] = (np.arange(out)[:, None] + np.arange(n_in)[None, :]) % 256
    nan = np.zeros(out, bool)
    nan[[3, 130, 255]] = True                                # NaN in these rows only
    w.codes[0, ~nan] = np.where((w.codes[0, ~nan] & 0x7F) == 0x7F, 0x30, w.codes[0, ~nan])
    w.scales[:], w.bits[:] = 1, 1
    wd = own.weight(w.tensor(dense=True))
    cols = (np.arange(T) * 37) % n_in
    codes = np.zeros((T, n_in), np.uint8)
    codes[np.arange(T), cols] = encode(1.0)
    bad = np.array([5, T - 2])
    codes[bad, [n_in - 1, 7]] = [0x7F, 0xFF]                 # NaN in two rows of x
    x = own.rows8(T, n_in, codes, np.full((T, nblocks(n_in)), 0x3F80, np.uint16))
    y = own.zeros(T * out if y_type == F32 else T * out // 2)
    with gpu.batch() as b:
        b.matmul_q8(wd, x, y, y_type)
    got = (gpu.read(y) if y_type == F32 else read_bf16(gpu, y)).reshape(T, out)
    fine = np.ones(T, bool)
    fine[bad] = False
    assert np.isnan(got[:, nan]).all() and np.isnan(got[bad]).all()
    assert np.array_equal(got[fine][:, ~nan], decode(w.codes[0])[:, cols].T[fine][:, ~nan])


@pytest.mark.parametrize("T,y_type", [(20, BF16), (5200, F32), (2600, BF16)])
def test_wide_scales_in_every_form(gpu, own, T, y_type):
    """Scales over 60 and 80 powers of two; NaN and infinite scales of a row and of
    a weight block, which reach their own outputs only."""
    rng = np.random.default_rng(T)
    n_in, out = 528, 384
    w = Weight8(rng, 1, out, n_in)
    w.bits[:] = (2.0 ** rng.integers(-60, 0, w.bits.shape)).astype(np.float32)
    w.bits[0, 1, 4], w.bits[0, 2, 0] = np.nan, np.inf
    w.scales[:] = w.bits
    codes, _ = random_rows(rng, T, n_in)
    bits = f32_to_bf16_bits((2.0 ** rng.integers(-40, 40, (T, 5))).astype(np.float32)).reshape(T, 5)
    bits[3, 1], bits[T - 1, 4] = 0x7FC0, 0x7F80
    wd, x = own.weight(w.tensor(dense=True)), own.rows8(T, n_in, codes, bits)
    y = own.zeros(T * out if y_type == F32 else T * out // 2)
    with gpu.batch() as b:
        b.matmul_q8(wd, x, y, y_type)
    got = (gpu.read(y) if y_type == F32 else read_bf16(gpu, y)).reshape(T, out).astype(np.float64)
    assert np.isnan(got[3]).all() and not np.isfinite(got[T - 1]).any()
    assert np.isnan(got[:, 128:256]).all() and not np.isfinite(got[:, 256:]).any()
    keep = [t for t in range(T) if t not in (3, T - 1)]
    with np.errstate(invalid="ignore"):
        values = w.value()[:128]
    check_rows(got[keep, :128], *product(rows_value(codes, bits)[keep], values), n_in, y_type == BF16)


@pytest.mark.parametrize("P", [30, 3000])
def test_swiglu_of_rows_that_are_not_finite(gpu, own, P):
    """A NaN code, a NaN and an infinite scale of a row, a NaN scale of a gate
    block: what they reach reads back as NaN, what they do not is whole."""
    rng = np.random.default_rng(P)
    n_in, ff = 272, 272
    gate, up = Weight8(rng, 1, ff, n_in), Weight8(rng, 1, ff, n_in)
    gate.bits[0, 1, 2] = np.nan
    gate.scales[:] = gate.bits
    codes, bits = random_rows(rng, P, n_in)
    bad = [4, 9, P - 1]
    codes[4, 271], bits[9, 1], bits[P - 1, 0] = 0x7F, 0x7FC0, 0x7F80
    gd, ud, x, q, ob = own.weight(gate.tensor()), own.weight(up.tensor()), own.rows8(P, n_in, codes, bits), own.rows8(P, ff), own.u32([0, P])
    with gpu.batch() as b:
        b.expert_swiglu_q8(gd, ud, x, ob, None, 1, q)
    c, s = gpu.read_rows8(q)
    v = rows_value(c, s)
    assert np.isnan(v[bad]).all() and np.isnan(v[:, 128:256]).all()
    keep = np.setdiff1d(np.arange(P), bad)
    with np.errstate(invalid="ignore"):
        want, dw = swiglu64(rows_value(codes, bits)[keep], gate, up, 0)
    for cols, blocks in ((slice(0, 128), slice(0, 1)), (slice(256, 272), slice(2, 3))):
        check_quantized(c[keep, cols], s[keep, blocks], want[:, cols], dw[:, cols])


@pytest.mark.parametrize("y_type", [F32, BF16])
def test_tiles_of_operands_just_under_four_gib(gpu, own, y_type):
    """Tiles address a matrix by 32-bit offsets: the last rows of 2^32 - 2^14
    codes of x, then of W."""
    rng = np.random.default_rng(14)
    n_in, many, few = 16384, (1 << 18) - 1, 96
    tail, tb = random_rows(rng, few, n_in)
    w = Weight8(rng, 1, 64, n_in)
    x = own.rows8(many, n_in)
    for b, a in zip(x.buffers, (tail, tb)):
        raw = a.reshape(-1).view(np.float32)
        gpu.write(b.view(len(b) - raw.size, raw.size), raw)
    wd, y = own.weight(w.tensor(dense=True)), own.zeros(many * 64 // (1 if y_type == F32 else 2), 0x55555555)
    with gpu.batch() as b:
        b.matmul_q8(wd, x, y, y_type)
    got = (gpu.read(y) if y_type == F32 else read_bf16(gpu, y)).reshape(many, 64)
    check_rows(got[-few:], *product(rows_value(tail, tb), w.value()), n_in, y_type == BF16)
    assert not got[:-few].any()
    # W: the rows of x of the same buffer, a scale of one for all
    t = Weight8(rng, 1, 1, 16).tensor(dense=True)
    t.dims = [n_in, many]
    wd = own.weight(t)
    scales = own.upload(np.ones(nblocks(many) * nblocks(n_in), np.float32))
    wd.c.data, wd.c.scales = x.c.codes, MoeRegionC(scales.ptr, 4 * len(scales))
    codes, bits = random_rows(rng, 40, n_in)
    rows, z = own.rows8(40, n_in, codes, bits), own.zeros(40 * many // (1 if y_type == F32 else 2), 0x55555555)
    with gpu.batch() as b:
        b.matmul_q8(wd, rows, z, y_type)
    got = (gpu.read(z) if y_type == F32 else read_bf16(gpu, z)).reshape(40, many)
    check_rows(got[:, -few:], *product(rows_value(codes, bits), decode(tail)), n_in, y_type == BF16)
    assert not got[:, :-few].any()


@pytest.mark.parametrize("T,n_in,out", [(2600, 16, 64), (2561, 1040, 130), (900, 2064, 770), (300, 256, 2500),
                                        (40, 128, 22000)])
@pytest.mark.parametrize("y_type", [F32, BF16])
def test_matmul_q8_of_many_rows(gpu, own, T, n_in, out, y_type):
    T = T * 2 if y_type == F32 else T    # (tiles start at twice the rows)
    rng = np.random.default_rng(T + n_in)
    w = Weight8(rng, 1, out, n_in)
    codes, bits = random_rows(rng, T, n_in)
    wd, x = own.weight(w.tensor(dense=True)), own.rows8(T, n_in, codes, bits)
    y = own.zeros(T * out if y_type == F32 else T * out // 2)
    with gpu.batch() as b:
        b.matmul_q8(wd, x, y, y_type)
    got = (gpu.read(y) if y_type == F32 else read_bf16(gpu, y)).reshape(T, out)
    check_rows(got, *product(rows_value(codes, bits), w.value()), n_in, y_type == BF16)


def test_more_tiles_than_a_block_lists_at_once(gpu, own):
    """256 blocks look their tiles up eight at a time: here each has nine or ten."""
    rng = np.random.default_rng(31)
    lens = [90000, 0, 7, 200, 179793]
    E, P, n_in = len(lens), sum(lens), 16
    w, w2 = Weight8(rng, E, 16, n_in), Weight8(rng, E, 16, n_in)
    codes, bits = random_rows(rng, P, n_in)
    offsets, perm = segments(rng, lens)
    wd, ud, x, y = own.weight(w.tensor()), own.weight(w2.tensor()), own.rows8(P, n_in, codes, bits), own.zeros(P * 8)
    ob, pb, q = own.u32(offsets), own.u32(perm), own.rows8(P, 16)
    with gpu.batch() as b:
        b.expert_matmul_q8(wd, x, ob, pb, y, BF16)
        b.expert_swiglu_q8(wd, ud, x, ob, pb, 1, q)
    got, (qc, qs) = read_bf16(gpu, y).reshape(P, 16)[perm], gpu.read_rows8(q)
    v = rows_value(codes, bits)
    for e in range(E):
        a, b_ = offsets[e], offsets[e + 1]
        if b_ > a:
            check_rows(got[a:b_], *product(v[a:b_], w.value(e)), n_in, True)
            check_quantized(qc[a:b_], qs[a:b_], *swiglu64(v[perm[a:b_]], w, w2, e))


@pytest.mark.parametrize("T", [1, 5, 20, 40])
@pytest.mark.parametrize("n_in", [8320, 16400])
def test_long_rows(gpu, own, T, n_in):
    """More blocks of 128 columns than the scales of one load."""
    rng = np.random.default_rng(T + n_in)
    w, w2 = Weight8(rng, 2, 48, n_in), Weight8(rng, 2, 48, n_in)
    codes, bits = random_rows(rng, T, n_in)
    wd, ud, x = own.weight(w.tensor()), own.weight(w2.tensor()), own.rows8(T, n_in, codes, bits)
    ob, y, z, q = own.u32([0, T // 2, T]), own.zeros(T * 48), own.zeros(T * 24), own.rows8(T, 48)
    with gpu.batch() as b:
        b.expert_matmul_q8(wd, x, ob, None, y)
        b.expert_matmul_q8(wd, x, ob, None, z, BF16)
        b.expert_swiglu_q8(wd, ud, x, ob, None, 1, q)
    v, (qc, qs) = rows_value(codes, bits), gpu.read_rows8(q)
    for e, r in enumerate((slice(0, T // 2), slice(T // 2, T))):
        if v[r].size:
            check_rows(gpu.read(y).reshape(T, 48)[r], *product(v[r], w.value(e)), n_in, False)
            check_rows(read_bf16(gpu, z).reshape(T, 48)[r], *product(v[r], w.value(e)), n_in, True)
            check_quantized(qc[r], qs[r], *swiglu64(v[r], w, w2, e))


@pytest.mark.parametrize("T", [3, 130, 3000])
def test_shared_expert_and_rows_named_twice(gpu, own, T):
    """One expert, no perm; then a perm that names rows more than once: each
    position reads the row it names, and each value of a result row named twice
    is that of one of its positions (which one may differ between the column
    tiles, whose blocks write in no set order)."""
    rng = np.random.default_rng(T)
    w, w2, dn = Weight8(rng, 1, 144, 256), Weight8(rng, 1, 144, 256), Weight8(rng, 1, 256, 144)
    codes, bits = random_rows(rng, T, 256)
    wd, ud, x, q = own.weight(w.tensor()), own.weight(w2.tensor()), own.rows8(T, 256, codes, bits), own.rows8(T, 144)
    dd, d3, y = own.weight(dn.tensor(dense=True)), own.weight(dn.tensor()), own.zeros(T * 128)
    ob, twice = own.u32([0, T]), rng.integers(0, T, T)
    pb, q2, y2 = own.u32(twice), own.rows8(T, 144), own.zeros(T * 128, 0x7FC07FC0)
    with gpu.batch() as b:
        b.expert_swiglu_q8(wd, ud, x, ob, None, 1, q)
        b.matmul_q8(dd, q, y, BF16)
        b.expert_swiglu_q8(wd, ud, x, ob, pb, 1, q2)
        b.expert_matmul_q8(d3, q, ob, pb, y2, BF16)
    qc, qs = gpu.read_rows8(q)
    check_quantized(qc, qs, *swiglu64(rows_value(codes, bits), w, w2, 0))
    got = read_bf16(gpu, y).reshape(T, 256)
    check_rows(got, *product(rows_value(qc, qs), dn.value()), 144, True)
    c2, s2 = gpu.read_rows8(q2)
    assert np.array_equal(c2, qc[twice]) and np.array_equal(s2, qs[twice])
    got2 = read_bf16(gpu, y2).reshape(T, 256)
    for row in range(T):
        at = np.flatnonzero(twice == row)
        assert np.isnan(got2[row]).all() if at.size == 0 else (got2[row] == got[at]).any(0).all()


@pytest.mark.parametrize("T,n_in,ff,E", [(1, 512, 512, 1), (10, 2048, 512, 10), (48, 512, 272, 4), (300, 256, 144, 2)])
def test_small_swiglu_over_and_over(gpu, own, T, n_in, ff, E):
    """The blocks that share a scale hand their rows to the last of them: the
    same bits in each of many calls in flight, by call and from a replayed graph,
    also after segments that overlap (more tiles than the launch has blocks for)."""
    rng = np.random.default_rng(T + ff)
    w, w2 = Weight8(rng, E, ff, n_in), Weight8(rng, E, ff, n_in)
    codes, bits = random_rows(rng, T, n_in)
    offsets = np.sort(np.r_[0, rng.integers(0, T + 1, E - 1), T])
    wd, ud, x, ob = own.weight(w.tensor()), own.weight(w2.tensor()), own.rows8(T, n_in, codes, bits), own.u32(offsets)
    over = own.u32(np.arange(E + 1) % 2 * T)
    many = [own.rows8(T, ff) for _ in range(24)]
    cap = gpu.capture()
    with cap as b:
        for q in many[:8]:
            b.expert_swiglu_q8(wd, ud, x, ob, None, 1, q)
    want, dw = (np.concatenate(v) for v in zip(*(swiglu64(rows_value(codes, bits)[a:c], w, w2, e)
                                                for e, (a, c) in enumerate(zip(offsets[:-1], offsets[1:])))))
    for turn in range(4):
        with gpu.batch() as b:
            b.expert_swiglu_q8(wd, ud, x, over, None, 1, many[23])
            b.graph(cap.graph)
            for q in many[8:]:
                b.expert_swiglu_q8(wd, ud, x, ob, None, 1, q)
        got = [gpu.read_rows8(q) for q in many]
        check_quantized(*got[0], want, dw)
        for c, s in got[1:]:
            assert np.array_equal(c, got[0][0]) and np.array_equal(s, got[0][1])
    cap.graph.destroy()


@pytest.mark.parametrize("T,n_in,ff", [(160, 2048, 512), (200, 1024, 512), (256, 1024, 512), (144, 1280, 528)])
@pytest.mark.parametrize("perm", [False, True])
def test_small_swiglu_after_more_tiles_than_a_launch_has(gpu, own, T, n_in, ff, perm):
    """Two segments of all rows hold more tiles than the launch has blocks for, and
    the cut falls inside a segment whose tiles go by panels of columns: each tile
    runs whole or not at all, so that the next call finds the counts at zero."""
    rng = np.random.default_rng(T + n_in)
    w, w2 = Weight8(rng, 3, ff, n_in), Weight8(rng, 3, ff, n_in)
    codes, bits = random_rows(rng, T, n_in)
    wd, ud, x = own.weight(w.tensor()), own.weight(w2.tensor()), own.rows8(T, n_in, codes, bits)
    offsets = [0, T // 3, T // 3, T]
    ob, over = own.u32(offsets), own.u32([0, T, 0, T])
    order = np.arange(T)
    if perm:
        order = rng.permutation(T)
    pb = own.u32(order) if perm else None
    many, spoilt = [own.rows8(T, ff) for _ in range(12)], own.rows8(T, ff)
    with gpu.batch() as b:
        for i, q in enumerate(many):
            if i % 3 == 1:
                b.expert_swiglu_q8(wd, ud, x, over, pb, 1, spoilt)
            b.expert_swiglu_q8(wd, ud, x, ob, pb, 1, q)
    v = rows_value(codes, bits)[order]
    want, dw = (np.concatenate(p) for p in zip(*(swiglu64(v[a:c], w, w2, e)
                                                for e, (a, c) in enumerate(zip(offsets[:-1], offsets[1:])))))
    first = gpu.read_rows8(many[0])
    check_quantized(*first, want, dw)
    for q in many[1:]:
        for i, j in zip(first, gpu.read_rows8(q)):
            assert np.array_equal(i, j)


@pytest.mark.parametrize("P,E,ff", [(2559, 1, 128), (1279, 1, 256), (2000, 47, 128), (2400, 34, 16), (106, 106, 16), (900, 26, 256)])
def test_the_largest_swiglus_in_two_launches(gpu, own, P, E, ff):
    """As many rows, and tiles, as the F32 rows and the list between the launches
    are for; one more of either goes in tiles of 128."""
    rng = np.random.default_rng(P)
    n_in = 144
    for P, E in ((P, E), (P + 1, E + 1)):
        w, w2 = Weight8(rng, E, ff, n_in), Weight8(rng, E, ff, n_in)
        offsets, perm = segments(rng, 1 + np.bincount(rng.integers(0, E, P - E), minlength=E))
        codes, bits = random_rows(rng, P, n_in)
        wd, ud, x, q = own.weight(w.tensor()), own.weight(w2.tensor()), own.rows8(P, n_in, codes, bits), own.rows8(P, ff)
        ob, pb = own.u32(offsets), own.u32(perm)
        with gpu.batch() as b:
            b.expert_swiglu_q8(wd, ud, x, ob, pb, 1, q)
        c, s = gpu.read_rows8(q)
        v = rows_value(codes, bits)[perm]
        for e in range(E):
            a, b_ = offsets[e], offsets[e + 1]
            if b_ > a:
                check_quantized(c[a:b_], s[a:b_], *swiglu64(v[a:b_], w, w2, e))


def test_more_tiles_than_32_bits_count(gpu, own):
    """8192 segments of all rows, 2^32 + 8192 tiles of 128: those of the first
    segments run, and with them every row has its product."""
    E, P, n_in, out = 16384, (1 << 26) + 128, 16, 2
    w = Weight8(np.random.default_rng(3), E, out, n_in)
    wd, x, y = own.weight(w.tensor()), own.rows8(P, n_in), own.zeros(P * out // 2)
    gpu.write(y, np.full(P * out // 2, 0x55555555, np.uint32).view(np.float32))
    ob = own.u32(np.arange(E + 1) % 2 * P)
    with gpu.batch() as b:
        b.expert_matmul_q8(wd, x, ob, None, y, BF16)
    assert not gpu.read_u32(y).any()


def test_two_gpus_at_once(gpu, own):
    """Batches of two engines on one device, both in flight: neither sees the
    other's rows on their way to 8 bits in a small SwiGLU."""
    rng = np.random.default_rng(17)
    T, n_in, ff, E = 48, 512, 512, 4
    w, w2 = Weight8(rng, E, ff, n_in), Weight8(rng, E, ff, n_in)
    second = Gpu(0)
    runs = []
    for g in (gpu, second):
        o = own if g is gpu else Owned(g)
        codes, bits = random_rows(rng, T, n_in)
        runs.append((g, o, o.weight(w.tensor()), o.weight(w2.tensor()), o.rows8(T, n_in, codes, bits),
                     o.u32([0, 10, 10, 31, T]), o.rows8(T, ff), o.rows8(T, ff)))
    for g, _, wd, ud, x, ob, q, _ in runs:
        with g.batch() as b:
            b.expert_swiglu_q8(wd, ud, x, ob, None, 1, q)
    batches = [Batch(g) for g, *_ in runs]
    for _ in range(50):
        for b, (_, _, wd, ud, x, ob, _, r) in zip(batches, runs):
            b.expert_swiglu_q8(wd, ud, x, ob, None, 1, r)
    for b in batches:
        b.finish()
    for g, o, _, _, _, _, q, r in runs:
        for i, j in zip(g.read_rows8(q), g.read_rows8(r)):
            assert np.array_equal(i, j)
    runs[1][1].release()


def test_rows_past_four_gib(gpu, own):
    """Row offsets that take more than 32 bits: the last rows of 4.3 GB of codes."""
    rng = np.random.default_rng(8)
    n_in, T, last = 8192, 524800, 96
    w, w2 = Weight8(rng, 1, 16, n_in), Weight8(rng, 1, 16, n_in)
    few, fb = random_rows(rng, 512, n_in)
    codes, bits = np.tile(few, (T // 512, 1)), np.tile(fb, (T // 512, 1))
    tail, tb = random_rows(rng, last, n_in)
    codes[-last:], bits[-last:] = tail, tb
    x, q, y, z = own.rows8(T, n_in, codes, bits), own.rows8(T, 16), own.zeros(T * 16), own.zeros(T * 8)
    wd, ud, dd, ob = own.weight(w.tensor()), own.weight(w2.tensor()), own.weight(w.tensor(dense=True)), own.u32([0, T])
    with gpu.batch() as b:
        b.expert_swiglu_q8(wd, ud, x, ob, None, 1, q)
        b.matmul_q8(dd, x, y)
        b.matmul_q8(dd, x, z, BF16)
    qc, qs = gpu.read_rows8(q)
    got, half = gpu.read(y).reshape(T, 16), read_bf16(gpu, z).reshape(T, 16)
    for r, c, s in ((slice(T - last, T), tail, tb), (slice(0, 512), few, fb), (slice(T - 1024, T - 512), few, fb)):
        v = rows_value(c, s)
        check_quantized(qc[r], qs[r], *swiglu64(v, w, w2, 0))
        check_rows(got[r], *product(v, w.value()), n_in, False)
        check_rows(half[r], *product(v, w.value()), n_in, True)


def test_norm_q8_of_more_rows_than_a_launch_is_wide(gpu, own):
    rng = np.random.default_rng(13)
    rows, n = (1 << 24) + 5, 16
    x, q = own.zeros(rows * n), own.rows8(rows, n)
    norm = own.weight(Tensor.dense([n], np.ones(n, np.float32)))
    at = [0, (1 << 22) - 1, 1 << 22, (1 << 24) - 1, rows - 1]
    v = rng.standard_normal((len(at), n)).astype(np.float32)
    for r, i in zip(v, at):
        gpu.write(x.view(i * n, n), r)
    with gpu.batch() as b:
        b.norm_q8(x, None, norm, None, None, q, 1e-6)
    c, s = gpu.read_rows8(q)
    want = norm64(v, np.ones(n), 1e-6)
    check_quantized(c[at], s[at], want, 70 * U * np.abs(want))
    rest = np.ones(rows, bool)
    rest[at] = False
    assert not c[rest].any() and np.all(s[rest] == 0x0080)   # the least scale, 2^-126


# -------------------------------------------------------------------- mix --
@pytest.mark.parametrize("T,K,h", [(1, 1, 16), (1, 10, 2048), (3, 8, 130), (5, 3, 7), (64, 10, 512), (300, 2, 1028)])
@pytest.mark.parametrize("x_type", [F32, BF16])
def test_mix_tokens(gpu, own, T, K, h, x_type):
    if x_type == BF16 and T * K * h % 2:
        pytest.skip("bf16 inputs come two to an element")
    rng = np.random.default_rng(T + K + h)
    x = rng.standard_normal((T, K, h)).astype(np.float32)
    if x_type == BF16:
        raw = f32_to_bf16_bits(x.ravel())
        x = bf16(raw).reshape(T, K, h)
        xb = own.upload(raw.view(np.float32))
    else:
        xb = own.upload(x)
    w = rng.standard_normal((T, K)).astype(np.float32)
    r = rng.standard_normal((T, h)).astype(np.float32)
    wb, rb, y = own.upload(w), own.upload(r), own.zeros(T * h)
    terms = x.astype(np.float64) * w.astype(np.float64)[..., None]
    want, mag = terms.sum(1), np.abs(terms).sum(1)
    with gpu.batch() as b:
        b.mix_tokens(xb, wb, None, y, T, x_type)
    plain = gpu.read(y).reshape(T, h)
    assert np.all(np.abs(plain - want) <= K * U * mag)
    with gpu.batch() as b:
        b.mix_tokens(xb, wb, rb, y, T, x_type)
        b.mix_tokens(xb, wb, rb, rb, T, x_type)      # the residual in place
    got = gpu.read(y).reshape(T, h)
    assert np.all(np.abs(got - (want + r)) <= (K + 1) * U * (mag + np.abs(r)))
    assert np.array_equal(gpu.read(rb).reshape(T, h), got)


def test_mix_tokens_equals_mix(gpu, own):
    rng = np.random.default_rng(4)
    T, K, h = 3, 5, 64
    x, w = own.upload(rng.standard_normal(T * K * h)), own.upload(rng.standard_normal(T * K))
    y, one = own.zeros(T * h), own.zeros(T * h)
    with gpu.batch() as b:
        b.mix_tokens(x, w, None, y, T)
        for t in range(T):
            b.mix(x.view(t * K * h, K * h), w.view(t * K, K), one.view(t * h, h))
    a, c = gpu.read(y), gpu.read(one)
    assert np.all(np.abs(a - c) <= 2 * K * U * 20)


# --------------------------------------------------------------- refusals --
def test_refusals(gpu, own):
    rng = np.random.default_rng(9)
    E, n_in, out, T = 3, 256, 64, 6
    wt, gt = Weight8(rng, E, out, n_in), Weight8(rng, 1, out, n_in)
    w3, w2 = own.weight(wt.tensor()), own.weight(gt.tensor(dense=True))
    codes, bits = random_rows(rng, T, n_in)
    x, y = own.rows8(T, n_in, codes, bits), own.zeros(T * out)
    q, ob, pb = own.rows8(T, out), own.u32([0, 2, 4, 6]), own.u32(np.arange(T))
    dense = own.weight(Tensor.dense([n_in, out], rng.standard_normal(n_in * out)))
    norm, xf = own.weight(Tensor.dense([n_in], np.ones(n_in, np.float32))), own.upload(np.ones(T * n_in))
    other = own.weight(Weight8(rng, E, out, n_in, BF16).tensor())

    def alter(w, **kw):
        c = type(w.c).from_buffer_copy(w.c)
        for k, v in kw.items():
            if k == "dims":
                for i, d in enumerate(v):
                    c.dims[i] = d
            else:
                setattr(c, k, v)
        return type(w)(c, w.regions, w.dims, 0)

    def rows(r, **kw):
        a = {"codes": r.c.codes, "scales": r.c.scales, "rows": r.rows, "n": r.n}
        a.update(kw)
        return Rows8(a["codes"], a["scales"], a["rows"], a["n"])

    short = MoeRegionC(x.c.codes.ptr, x.c.codes.bytes - 1)
    odd = MoeRegionC(x.c.codes.ptr + 4, (T - 1) * n_in)
    foreign = MoeRegionC(0x1000, x.c.codes.bytes)
    bad = [
        lambda b: b.matmul_q8(dense, x, y),
        lambda b: b.matmul_q8(w3, x, y),
        lambda b: b.matmul_q8(alter(w2, group_size=64), x, y),
        lambda b: b.matmul_q8(alter(w2, scale_type=7), x, y),
        lambda b: b.matmul_q8(alter(w2, dims=[n_in, out + 1]), x, y),
        lambda b: b.matmul_q8(alter(w2, dims=[n_in // 2 - 8, 2 * out]), x, y),
        lambda b: b.matmul_q8(alter(w2, dims=[0, out]), x, y),
        lambda b: b.matmul_q8(w2, rows(x, n=128, rows=2 * T), y),
        lambda b: b.matmul_q8(w2, rows(x, rows=T - 1), y),
        lambda b: b.matmul_q8(w2, rows(x, rows=0), y),
        lambda b: b.matmul_q8(w2, rows(x, codes=short), y),
        lambda b: b.matmul_q8(w2, rows(x, codes=foreign), y),
        lambda b: b.matmul_q8(w2, rows(x, codes=odd, rows=T - 1,
                                       scales=MoeRegionC(x.c.scales.ptr, (T - 1) * 4)), y.view(0, (T - 1) * out)),
        lambda b: b.matmul_q8(w2, x, y.view(0, T * out - 1)),
        lambda b: b.matmul_q8(w2, x, y, BF16),
        lambda b: b.matmul_q8(w2, x, y, F16),
        lambda b: b.matmul_q8(w2, x, Buffer(gpu, MoeBufferC(w2.c.data.ptr, T * out), 0)),
        lambda b: b.matmul(w2, xf, y, T),                       # the F32 op takes no 8-bit weights
        lambda b: b.expert_matmul_q8(w2, x, ob, pb, y),
        lambda b: b.expert_matmul_q8(w3, x, ob.view(0, 3), pb, y),
        lambda b: b.expert_matmul_q8(w3, x, ob, pb.view(0, T - 1), y),
        lambda b: b.expert_swiglu_q8(w3, other, x, ob, pb, 1, q),
        lambda b: b.expert_swiglu_q8(w3, alter(w3, dims=[n_in, out - 1, E]), x, ob, pb, 1, q),
        lambda b: b.expert_swiglu_q8(w3, w3, x, ob, pb, 2, q),
        lambda b: b.expert_swiglu_q8(w3, w3, x, ob, pb, 0, q),
        lambda b: b.expert_swiglu_q8(w3, w3, x, ob, None, 2, q),
        lambda b: b.expert_swiglu_q8(w3, w3, x, ob, pb, 1, x),
        lambda b: b.norm_q8(xf, None, w2, None, None, x, 1e-6),
        lambda b: b.norm_q8(xf, None, norm, None, None, x, 0.0),
        lambda b: b.norm_q8(xf, None, norm, None, None, x, float("nan")),
        lambda b: b.norm_q8(xf, None, norm, None, xf, x, 1e-6),
        lambda b: b.norm_q8(xf.view(0, n_in), None, norm, None, None, x, 1e-6),
        lambda b: b.norm_q8(xf, xf.view(0, n_in), norm, None, None, x, 1e-6),
        lambda b: b.norm_q8(xf, None, norm, y, None, x, 1e-6),
        lambda b: b.mix_tokens(xf, y.view(0, T), None, y.view(0, T * n_in // 8), T),
        lambda b: b.mix_tokens(xf, y.view(0, T), None, xf, T),
        lambda b: b.mix_tokens(xf, y.view(0, T), None, y, 0),
        lambda b: b.mix_tokens(xf, y.view(0, T + 1), None, y, T),
        lambda b: b.mix_tokens(xf, y.view(0, T), None, y, T, F16),
    ]
    before = gpu.read(y).copy()
    for i, f in enumerate(bad):
        b = Batch(gpu)
        try:
            with pytest.raises(ShapeError):
                f(b)
                print("not refused:", i)
        finally:
            b.finish()
    assert np.array_equal(gpu.read(y), before)
    # outside of a batch
    b = Batch(gpu, begin=False)
    with pytest.raises(ShapeError):
        b.matmul_q8(w2, x, y)


def test_lengths_past_the_address_space_are_refused(gpu, own):
    """2^62 + 4 elements are 16 bytes in 64 bits: not those of an allocation."""
    a, b_ = own.zeros(64), own.zeros(64)
    for n in ((1 << 62) + 4, (1 << 63) + 4, (1 << 64) - 8):
        long, other = (Buffer(gpu, MoeBufferC(x.ptr + 32, n), x.ptr) for x in (a, b_))
        with pytest.raises(ShapeError):
            gpu.clear(long)
        with gpu.batch() as b:
            for f in (lambda: b.copy(long, other), lambda: b.add(long, other, long),
                      lambda: b.mix_tokens(long, long, None, other, n)):
                with pytest.raises(ShapeError):
                    f()


# ------------------------------------------------------------------ chain --
def chain(b, o, d):
    """One MoE block over T tokens by the operators."""
    b.norm_q8(d["x"], d["r"], d["norm"], d["sum"], d["xn"], d["x8"], 1e-6)
    b.matmul(d["router"], d["xn"], d["logits"], d["T"])
    b.route_tokens(d["logits"], d["ids"], d["w"], d["T"], True)
    b.dispatch(d["ids"], d["T"], d["K"], d["E"], d["counts"], d["offsets"], d["perm"], d["pos"])
    b.expert_swiglu_q8(d["gate"], d["up"], d["x8"], d["offsets"], d["perm"], d["K"], d["a8"])
    b.expert_matmul_q8(d["down"], d["a8"], d["offsets"], d["perm"], d["y"], d["ytype"])
    b.mix_tokens(d["y"], d["w"], d["sum"], d["out"], d["T"], d["ytype"])


def chain_state(own, rng, T, h, E, K, ff, ytype):
    d = {"T": T, "K": K, "E": E, "ytype": ytype}
    d["host"] = {n: Weight8(rng, E, *s) for n, s in (("gate", (ff, h)), ("up", (ff, h)), ("down", (h, ff)))}
    for n, w in d["host"].items():
        d[n] = own.weight(w.tensor())
    d["hx"], d["hr"] = (rng.standard_normal((T, h)).astype(np.float32) for _ in range(2))
    d["x"], d["r"] = own.upload(d["hx"]), own.upload(d["hr"])
    d["hn"] = (1 + 0.1 * rng.standard_normal(h)).astype(np.float32)
    d["norm"] = own.weight(Tensor.dense([h], d["hn"]))
    d["router"] = own.weight(Tensor.dense([h, E], rng.standard_normal(h * E) * 0.05))
    for n, s in (("sum", T * h), ("xn", T * h), ("logits", T * E), ("ids", T * K), ("w", T * K), ("counts", E),
                 ("offsets", E + 1), ("perm", T * K), ("pos", T * K), ("out", T * h),
                 ("y", T * K * h // (2 if ytype == BF16 else 1))):
        d[n] = own.zeros(s)
    d["x8"], d["a8"] = own.rows8(T, h), own.rows8(T * K, ff)
    return d


@pytest.mark.parametrize("T,h,E,K,ff,ytype", [(1, 256, 8, 2, 128, F32), (7, 272, 5, 3, 48, F32),
                                              (70, 256, 6, 4, 144, BF16), (200, 128, 4, 2, 256, BF16),
                                              (700, 256, 6, 4, 144, BF16), (1300, 128, 5, 4, 128, F32)])
def test_chain(gpu, own, T, h, E, K, ff, ytype):
    """The operators as a block uses them, each stage against 64 bits over what
    the stage before it wrote; then captured and replayed over new inputs."""
    rng = np.random.default_rng(T * 7 + h)
    d = chain_state(own, rng, T, h, E, K, ff, ytype)
    with gpu.batch() as b:
        chain(b, own, d)

    def check():
        s = d["hx"] + d["hr"]
        assert np.array_equal(gpu.read(d["sum"]).reshape(T, h), s)
        xn = norm64(s, d["hn"].astype(np.float64), 1e-6)
        check_quantized(*gpu.read_rows8(d["x8"]), xn, 70 * U * np.abs(xn))
        off, perm = gpu.read_u32(d["offsets"]), gpu.read_u32(d["perm"])
        ids, w = gpu.read_u32(d["ids"]).reshape(T, K), gpu.read(d["w"]).reshape(T, K).astype(np.float64)
        assert off[E] == T * K
        x = rows_value(*gpu.read_rows8(d["x8"]))
        a8 = gpu.read_rows8(d["a8"])
        a = rows_value(*a8)
        want, dw = np.zeros((T * K, ff)), np.zeros((T * K, ff))
        y, ym, yg = (np.zeros((T * K, h)) for _ in range(3))
        for e in range(E):
            p = np.arange(off[e], off[e + 1])
            assert np.array_equal(ids.ravel()[perm[p]], np.full(p.size, e))
            if p.size:
                want[p], dw[p] = swiglu64(x[perm[p] // K], d["host"]["gate"], d["host"]["up"], e)
                y[perm[p]], ym[perm[p]], yg[perm[p]] = product(a[p], d["host"]["down"].value(e))
        check_quantized(*a8, want, dw)
        got = (read_bf16(gpu, d["y"]) if ytype == BF16 else gpu.read(d["y"]).astype(np.float64)).reshape(T * K, h)
        check_rows(got, y, ym, yg, ff, ytype == BF16)
        terms = got.reshape(T, K, h) * w[..., None]
        out = terms.sum(1) + s
        assert np.all(np.abs(gpu.read(d["out"]).reshape(T, h) - out) <= (K + 1) * U * (np.abs(terms).sum(1) + np.abs(s)))

    check()
    cap = gpu.capture()
    with cap as b:
        chain(b, own, d)
    for _ in range(3):
        d["hx"] = rng.standard_normal((T, h)).astype(np.float32)
        gpu.write(d["x"], d["hx"])
        with gpu.batch() as b:
            b.graph(cap.graph)
        check()
        first = [gpu.read(d[n]).copy() for n in ("out", "y")] + list(gpu.read_rows8(d["a8"]))
        with gpu.batch() as b:
            chain(b, own, d)
        again = [gpu.read(d[n]) for n in ("out", "y")] + list(gpu.read_rows8(d["a8"]))
        for i, j in zip(first, again):
            assert np.array_equal(np.asarray(i).view(np.uint8), np.asarray(j).view(np.uint8))
    cap.graph.destroy()
