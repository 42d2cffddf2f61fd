"""The 8-bit floating point operators' plain forms and host side, on the CPU."""
import ctypes as C

import numpy as np
import pytest

from helpers_q8 import POS, TABLE, Weight8, decode, encode, nblocks, quantize_rows, random_rows, rows_value
from hip_backend import BF16, E4M3, F16, F32, Buffer, Gpu, Rows8, ShapeError, Weight, api


def test_e4m3_codes_round_to_nearest_even():
    codes = np.arange(256, dtype=np.uint8)
    real = (codes & 0x7F) != 0x7F
    assert np.array_equal(encode(decode(codes[real])), codes[real])
    assert POS[-1] == 448 and POS[1] == 2.0 ** -9 and np.all(np.diff(POS) > 0)
    for a, b, even in zip(POS[:-1], POS[1:], range(126)):
        want = even if even % 2 == 0 else even + 1
        assert encode((a + b) / 2) == want
        assert encode(np.nextafter((a + b) / 2, 1e9)) == even + 1
    assert encode(464.0) == 0x7E and np.isnan(TABLE[encode(465.0)]) and np.isnan(TABLE[encode(np.nan)])


def test_quantized_rows_read_back_within_half_a_step():
    rng = np.random.default_rng(3)
    y = rng.standard_normal((5, 272)).astype(np.float32)
    y[1] = 0
    y[2, :128] *= np.float32(1e-42)
    codes, bits = quantize_rows(y)
    got = rows_value(codes, bits)
    assert np.all(np.abs(got - y)[[0, 2, 3, 4]] <= np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * np.abs(y).max())[[0, 2, 3, 4]])
    assert np.all(got[1] == 0)
    y[3, 200] = np.inf
    y[4, 5] = np.nan
    codes, bits = quantize_rows(y)
    got = rows_value(codes, bits)
    assert np.isnan(got[3, 128:256]).all() and np.isfinite(got[3, :128]).all() and np.isfinite(got[3, 256:]).all()
    assert np.isnan(got[4, :128]).all() and np.isfinite(got[4, 128:]).all()


def test_entries_without_a_gpu_are_refused():
    lib = api.load_library()
    w, r, b = api.MoeWeightC(), api.MoeRows8C(), api.MoeBufferC()
    assert lib.moe_norm_q8(None, b, b, C.byref(w), b, b, r, 1e-6) == 3
    assert lib.moe_matmul_q8(None, C.byref(w), r, b, 0) == 3
    assert lib.moe_expert_swiglu_q8(None, C.byref(w), C.byref(w), r, b, b, 1, r) == 3
    assert lib.moe_expert_matmul_q8(None, C.byref(w), r, b, b, b, 0) == 3
    assert lib.moe_mix_tokens(None, b, 0, b, b, b, 1) == 3


def test_block8_tensors_hold_codes_and_block_scales():
    rng = np.random.default_rng(1)
    for st, size in ((F32, 4), (F16, 2), (BF16, 2)):
        w = Weight8(rng, 3, 130, 272, st)
        t = w.tensor()
        assert t.dims == [272, 130, 3] and t.dtype == E4M3 and t.bits == 0 and t.group_size == 128
        assert t.data.nbytes == 3 * 130 * 272 and t.scales.nbytes == 3 * 2 * 3 * size
        assert w.value(2).shape == (130, 272) and nblocks(272) == 3
    codes, bits = random_rows(rng, 4, 48)
    assert codes.shape == (4, 48) and bits.shape == (4, 1)


class Memory:
    """Takes a Gpu's writes on the host."""

    write_rows8 = Gpu.write_rows8

    def __init__(self):
        self.written = []

    def zeros(self, n):
        return Buffer(None, api.MoeBufferC(0x1000, n), 0x1000)

    def write(self, b, a):
        self.written.append(a.view(np.uint8))


def test_rows8_are_written_whole_or_refused():
    rows, n = 3, 272
    codes, bits = np.ones((rows, n), np.uint8), np.ones((rows, 3), np.uint16)
    m = Memory()
    r = Gpu.rows8(m, rows, n)
    for c, s in ((codes[:2], bits), (codes, bits[:2]), (codes, bits[:, :2]), (codes[:, :-16], bits), (codes, None),
                 (None, bits), (np.ones((rows + 1, n), np.uint8), bits), (codes, np.ones((rows, 4), np.uint16))):
        with pytest.raises(ShapeError):
            Gpu.write_rows8(m, r, c, s)
        with pytest.raises(ShapeError):
            Gpu.rows8(m, rows, n, c, s)
    own = Rows8(api.MoeRegionC(), api.MoeRegionC(), rows, n)      # regions that the caller holds
    with pytest.raises(ShapeError):
        Gpu.write_rows8(m, own, codes, bits)
    with pytest.raises(ShapeError):
        Gpu.read_rows8(m, own)
    assert not m.written
    Gpu.write_rows8(m, r, codes, bits)
    assert [a.size for a in m.written] == [816, 20] and m.written[0].all() and m.written[1][:18:2].all()


def test_reshaped_weights_keep_the_blocks_of_their_scales():
    def weight(dims, dtype=E4M3):
        c = api.MoeWeightC()
        c.dtype, c.ndims = dtype, len(dims)
        c.dims[:len(dims)] = dims
        return Weight(c, [], dims, 0)

    for dims, to in (([272, 130], [272, 130, 1]), ([272, 130, 1], [272, 130]), ([272, 256, 3], [272, 768]),
                     ([272, 768], [272, 256, 3]), ([272, 256, 3], [272, 384, 2])):
        r = weight(dims).reshape(to)
        assert r.dims == to and list(r.c.dims[:len(to)]) == to and r.c.ndims == len(to)
    for dims, to in (([256, 256], [512, 128]), ([272, 130, 4], [272, 520]), ([272, 520], [272, 130, 4]),
                     ([272, 192, 2], [272, 128, 3]), ([256, 128], [256 * 128]), ([16, 4, 2], [16, 8])):
        with pytest.raises(ShapeError):
            weight(dims).reshape(to)
        assert weight(dims, F32).reshape(to).dims == to
