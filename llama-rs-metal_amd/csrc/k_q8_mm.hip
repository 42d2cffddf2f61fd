// Products of 8-bit rows with block-scaled 8-bit weights, dense and grouped by
// expert over ragged segments:
//
//   y[t, o] = sum over blocks b of 128 columns of
//             sx[t, b] * sw[o / 128, b] * sum_{k in b} x[t, k] * w[o, k]
//
// A block's inner sum runs on the matrix cores over the bare codes; its two
// scales multiply it in F32 as it joins the running sum.
//
// Two inner products, by what the output keeps:
//  - F32 outputs: the codes become f16 (exact) and go to
//    v_mfma_f32_16x16x32_f16, whose sums are F32's.
//  - bf16 and 8-bit outputs: v_mfma_f32_16x16x128_f8f6f4 on the codes
//    themselves, twice the rate.  It aligns eight products at a time to the
//    largest of them and cuts them at 2^-13 of its power of two before the F32
//    sum: 1.7e-5 off in 2-norm for normal data, where the output's own
//    rounding is 1.7e-3 (bf16) or 2.3e-2 (8 bits).
//
// Operand layout of both: the weight rows are the matrix instruction's rows
// (operand A), the tokens its columns (B).  Lane l = 16q + c holds row c's (token c's)
// bytes 16q .. 16q + 15 and 64 + 16q .. 64 + 16q + 15 of a block of 128, the
// same permutation of the columns on both sides; the result's lane 16q + c
// holds token c and four rows 4q + i.  A wave owns 64 weight rows as four
// row tiles whose rows interleave, so that a lane's results over its tiles are
// neighbouring outputs of one token.
#include "q8.hpp"

namespace moehip {

namespace q8 {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256, kWaves = 4;
constexpr int kWaveRows = 64;                     // weight rows per wave
constexpr int kBlockRows = kWaveRows * kWaves;    // and per block

enum { SWIGLU = 0, F32OUT = 1, BF16OUT = 2 };

struct Args {
    const uint8_t *w, *w2;        // codes (w2: the up weights of SWIGLU)
    const void *ws, *ws2;         // block scales, of type `stype`
    const uint8_t *x;             // input rows' codes [xrows, in]
    const uint16_t *xs;           // and scales [xrows, kb]
    const uint32_t *offsets;      // [experts + 1], or null: one segment of all positions
    const uint32_t *perm;         // [P] pair of each position, or null: the position itself
    void *y;                      // F32OUT / BF16OUT: [P, out]
    uint8_t *codes;               // SWIGLU: [P, out] and scales [P, ceil(out / 128)]
    uint16_t *scales;
    uint32_t stype, xrows, in, out, kb, experts, P, kdiv;
    uint32_t col_tiles;           // tiles along the outputs
};

// The work of this block: one of the M-tiles (runs of BM positions of a segment,
// experts ascending) times one column tile.  Workgroup b runs on XCD b % 8; the
// items are split into eight contiguous ranges, one per XCD, so the tiles that
// share an expert's weights and a run's rows meet in one L2.  Every thread of the
// block calls it; false (for all) where there is no item left.  Offsets past P
// count as P and a segment that ends before it starts is empty.
struct Tile {
    uint32_t e, m0, end, ct;
};
constexpr uint32_t kXcds = 8;
template <int BM>
__device__ __forceinline__ bool find_tile(const Args &a, Tile &t, uint32_t *lds /* 8 words */) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const uint32_t per = (a.experts + kThreads - 1) / kThreads, e0 = tid * per;
    auto seg = [&](uint32_t e, uint32_t &lo, uint32_t &n) {
        lo = min(a.offsets[e], a.P);
        const uint32_t hi = min(a.offsets[e + 1], a.P);
        n = hi > lo ? (hi - lo + BM - 1) / BM : 0u;
        return hi;
    };
    uint32_t mine = 0, before = 0, total = (a.P + BM - 1) / BM;
    if (a.offsets) {
        for (uint32_t i = 0; i < per && e0 + i < a.experts; i++) {
            uint32_t lo, n;
            seg(e0 + i, lo, n);
            mine += n;
        }
        uint32_t incl = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(incl, d);
            if ((int)lane >= d) incl += up;
        }
        if (lane == 63) lds[wv] = incl;
        __syncthreads();
        before = incl - mine;
        for (uint32_t v = 0; v < wv; v++) before += lds[v];
        total = lds[0] + lds[1] + lds[2] + lds[3];
    }
    const uint64_t items = (uint64_t)total * a.col_tiles, range = (items + kXcds - 1) / kXcds;
    const uint64_t item = blockIdx.x % kXcds * range + blockIdx.x / kXcds;
    if (blockIdx.x / kXcds >= range || item >= items) return false;
    const uint32_t tile = (uint32_t)(item / a.col_tiles);
    t.ct = (uint32_t)(item - (uint64_t)tile * a.col_tiles);
    if (!a.offsets) {
        t.e = 0, t.m0 = tile * BM, t.end = min(a.P, t.m0 + BM);
        return true;
    }
    if (tile >= before && tile < before + mine) {
        for (uint32_t i = 0; i < per && e0 + i < a.experts; i++) {
            uint32_t lo, n;
            const uint32_t hi = seg(e0 + i, lo, n);
            if (tile - before < n) {
                lds[4] = e0 + i;
                lds[5] = lo + (tile - before) * BM;
                lds[6] = hi;
                break;
            }
            before += n;
        }
    }
    __syncthreads();
    t.e = __builtin_amdgcn_readfirstlane(lds[4]);
    t.m0 = __builtin_amdgcn_readfirstlane(lds[5]);
    t.end = min(__builtin_amdgcn_readfirstlane(lds[6]), t.m0 + BM);
    return true;
}

__device__ __forceinline__ float scale_at(const void *p, uint32_t type, uint64_t i) {
    return type == 0 ? load_scalar<0>(p, i) : type == 1 ? load_scalar<1>(p, i) : load_scalar<30>(p, i);
}

__device__ __forceinline__ h8 f16_of(uint32_t lo, uint32_t hi) {
    const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, false);
    const h2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, true);
    const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, false);
    const h2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, true);
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A lane's 32 codes of one row and block.
struct Codes {
    u32x4q lo, hi;
    __device__ __forceinline__ i32x8 all() const {
        return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    }
};
template <bool F16>
struct Operand;
template <>
struct Operand<false> {
    i32x8 v;
    __device__ __forceinline__ explicit Operand(const Codes &c) : v(c.all()) {}
};
template <>
struct Operand<true> {
    h8 v[4];
    __device__ __forceinline__ explicit Operand(const Codes &c)
        : v{f16_of(c.lo[0], c.lo[1]), f16_of(c.lo[2], c.lo[3]), f16_of(c.hi[0], c.hi[1]), f16_of(c.hi[2], c.hi[3])} {}
};
__device__ __forceinline__ f32x4q block_dot(const Operand<false> &a, const Operand<false> &b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, f32x4q{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4q block_dot(const Operand<true> &a, const Operand<true> &b) {
    f32x4q c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; s++) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[s], b.v[s], c, 0, 0, 0);
    return c;
}

// The outputs of a wave's 64 weight rows (from n0) for NS token tiles: acc[j][i]
// holds row tile j, token tile i; to[i] is where the lane's token of tile i goes.
template <int MODE, int NS, int TT>
__device__ __forceinline__ void store_tile(const Args &a, const f32x4q (&acc)[4][NS], const uint32_t (&to)[NS],
                                           uint32_t n0, uint32_t ct, uint32_t wv, uint32_t *tops) {
    constexpr int BM = 16 * TT;
    const uint32_t lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4, ob = (a.out + 127) / 128;
    if constexpr (MODE == SWIGLU) {
        const uint32_t col = n0 + 8 * q;
        const bool cols_in = col < a.out;  // (out is a multiple of 16: all eight columns or none)
        float act[NS][8];
#pragma unroll
        for (int i = 0; i < NS; i++) {
            uint32_t top = 0;
#pragma unroll
            for (int r = 0; r < 8; r++) {
                const float g = acc[r / 4][i][r % 4], u = acc[2 + r / 4][i][r % 4];
                act[i][r] = g / (1.0f + expf(-g)) * u;
                if (cols_in) top = max(top, abs_word(act[i][r]));
            }
            top = max_xor32_u(max_xor16_u(top));
            if (q == 0) tops[wv * BM + 16 * i + c] = top;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NS; i++) {
            const uint32_t at = 16 * i + c;
            const uint32_t sb = q8_scale_bits(max(max(tops[at], tops[BM + at]), max(tops[2 * BM + at], tops[3 * BM + at])));
            if (to[i] == 0xffffffffu) continue;
            const float r = 1.0f / bf16_to_f32(sb);
            if (cols_in)
                *reinterpret_cast<u32x2q *>(a.codes + (uint64_t)to[i] * a.out + col) =
                    u32x2q{q8_codes4(act[i][0], act[i][1], act[i][2], act[i][3], r),
                           q8_codes4(act[i][4], act[i][5], act[i][6], act[i][7], r)};
            if (wv == 0 && q == 0) a.scales[(uint64_t)to[i] * ob + ct] = (uint16_t)sb;
        }
    } else {
        const uint32_t col = n0 + 16 * q;
        // whole groups of four where every row starts aligned
        const bool vec = a.out % 4 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15u) == 0;
#pragma unroll
        for (int i = 0; i < NS; i++) {
            if (to[i] == 0xffffffffu) continue;
            const uint64_t at = (uint64_t)to[i] * a.out + col;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const f32x4q v = acc[j][i];
                const uint32_t cj = col + 4 * j;
                if constexpr (MODE == F32OUT) {
                    float *y = static_cast<float *>(a.y) + at + 4 * j;
                    if (vec) {
                        if (cj < a.out) *reinterpret_cast<f32x4q *>(y) = v;
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (cj + r < a.out) y[r] = v[r];
                    }
                } else {
                    uint16_t *y = static_cast<uint16_t *>(a.y) + at + 4 * j;
                    uint32_t b[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) b[r] = bf16_bits(v[r]);
                    if (vec) {
                        if (cj < a.out) *reinterpret_cast<u32x2q *>(y) = u32x2q{b[0] | b[1] << 16, b[2] | b[3] << 16};
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (cj + r < a.out) y[r] = (uint16_t)b[r];
                    }
                }
            }
        }
    }
}

// TT: token tiles of 16 per block.
template <int MODE, int TT>
__global__ __launch_bounds__(kThreads) void mm_kernel(Args a) {
    constexpr bool kF16 = MODE == F32OUT;
    constexpr int BM = 16 * TT;
    __shared__ uint32_t lds[8];
    __shared__ uint32_t tops[MODE == SWIGLU ? kWaves * BM : 1];
    Tile t;
    if (!find_tile<BM>(a, t, lds)) return;
    const uint32_t ct = t.ct;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, c = lane & 15, q = lane >> 4;
    // the wave's rows: SWIGLU 32 gate and 32 up rows of one run of 32 outputs
    const uint32_t n0 = MODE == SWIGLU ? ct * (kBlockRows / 2) + wv * 32 : ct * kBlockRows + wv * kWaveRows;
    const uint8_t *wrow[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t r = MODE == SWIGLU ? n0 + 8 * (c >> 2) + 4 * (j & 1) + (c & 3) : n0 + 16 * (c >> 2) + 4 * j + (c & 3);
        const uint8_t *base = MODE == SWIGLU && j >= 2 ? a.w2 : a.w;
        wrow[j] = base + ((uint64_t)t.e * a.out + min(r, a.out - 1)) * a.in;  // rows past `out` are not stored
    }
    const uint32_t ob = (a.out + 127) / 128;
    const uint64_t srow = ((uint64_t)t.e * ob + min(n0 / 128, ob - 1)) * a.kb;
    // the lane's tokens (positions past the segment's end repeat its first row and are not stored)
    const uint8_t *xrow[TT];
    const uint16_t *xsrow[TT];
    uint32_t to[TT];  // where the position's outputs go: a row, or 0xffffffff for nowhere
#pragma unroll
    for (int i = 0; i < TT; i++) {
        const uint32_t p = t.m0 + 16 * i + c;
        const bool live = p < t.end;
        const uint32_t pair = a.perm ? a.perm[live ? p : t.m0] : (live ? p : t.m0);
        uint32_t row;
        if (MODE == SWIGLU) {
            row = pair / a.kdiv;
            to[i] = live && row < a.xrows ? p : 0xffffffffu;
        } else {
            row = live ? p : t.m0;
            to[i] = live && pair < a.P ? pair : 0xffffffffu;
        }
        row = min(row, a.xrows - 1);
        xrow[i] = a.x + (uint64_t)row * a.in;
        xsrow[i] = a.xs + (uint64_t)row * a.kb;
    }
    f32x4q acc[4][TT] = {};
    for (uint32_t kb = 0; kb < a.kb; kb++) {
        const uint32_t k = kb * 128 + 16 * q;
        // columns past `in`: the weights' codes are zero, the tokens' any of the row
        const bool lo_in = k < a.in, hi_in = k + 64 < a.in;
        const uint32_t klo = lo_in ? k : 0, khi = hi_in ? k + 64 : 0;
        Codes wc[4], xc[TT];
        const u32x4q zero = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            wc[j].lo = *reinterpret_cast<const u32x4q *>(wrow[j] + klo);
            wc[j].hi = *reinterpret_cast<const u32x4q *>(wrow[j] + khi);
            if (!lo_in) wc[j].lo = zero;
            if (!hi_in) wc[j].hi = zero;
        }
        float sx[TT];
#pragma unroll
        for (int i = 0; i < TT; i++) {
            const uint32_t klast = kb * 128;  // (a row's codes past `in` are replaced by ones of this block)
            xc[i].lo = *reinterpret_cast<const u32x4q *>(xrow[i] + (lo_in ? k : klast));
            xc[i].hi = *reinterpret_cast<const u32x4q *>(xrow[i] + (hi_in ? k + 64 : klast));
            sx[i] = bf16_to_f32(xsrow[i][kb]);
        }
        const float sw = scale_at(a.ws, a.stype, srow + kb);
        const float sw2 = MODE == SWIGLU ? scale_at(a.ws2, a.stype, srow + kb) : sw;
#pragma unroll
        for (int i = 0; i < TT; i++) {
            const Operand<kF16> xo(xc[i]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const f32x4q d = block_dot(Operand<kF16>(wc[j]), xo);
                const float s = sx[i] * (MODE == SWIGLU && j >= 2 ? sw2 : sw);
#pragma unroll
                for (int r = 0; r < 4; r++) acc[j][i][r] = fmaf(d[r], s, acc[j][i][r]);
            }
        }
    }
    store_tile<MODE, TT, TT>(a, acc, to, n0, ct, wv, tops);
}

// The same product for many rows per expert: a block of 128 (64 for F32 outputs)
// tokens.  The token rows of a block of 128 columns reach LDS by buffer DMA
// (eight rows of 128 bytes an instruction, 16-byte chunks XOR-swizzled by half
// the row number so that 16 rows' equal chunks lie in distinct banks), double
// buffered, one barrier a step; the weights go from memory straight to the
// waves' registers, one step ahead (no two waves share a weight row).  The
// rows' and weights' scales of 16 steps wait in LDS as F32.
typedef __attribute__((address_space(3))) void *lds_ptr;
constexpr int kGroup = 16;  // steps whose scales are in LDS together

template <int BM>
struct TileLds {
    uint8_t x[2][BM * 128];
    float sx[2][kGroup][BM];
    float sw[2][2][kGroup];
    uint32_t tops[kWaves * BM];
    uint32_t find[8];
};

template <int MODE, int TT, int NS>
__device__ __forceinline__ void tile_body(const Args &a, const Tile &t, TileLds<16 * TT> &lds) {
    constexpr bool kF16 = MODE == F32OUT;
    constexpr int BM = 16 * TT, ND = NS / 2;  // ND: DMA instructions a wave issues per step
    static_assert(NS % 2 == 0, "32 rows a round of DMA");
    const uint32_t tid = threadIdx.x, lane = tid & 63, c = lane & 15, q = lane >> 4;
    const uint32_t wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n0 = MODE == SWIGLU ? t.ct * (kBlockRows / 2) + wv * 32 : t.ct * kBlockRows + wv * kWaveRows;
    const uint32_t nb = min(n0, a.out - 1);
    const uint32_t nk = a.kb, tail = a.in % 128;
    // weights: one resource per matrix from row nb on, a lane's four rows as offsets
    const uint64_t wbase = ((uint64_t)t.e * a.out + nb) * a.in;
    const uint32_t wbytes = (uint32_t)min((uint64_t)(a.out - nb) * a.in, (uint64_t)0xffffffffu);
    const __amdgpu_buffer_rsrc_t rw = buffer_rsrc(a.w + wbase, wbytes);
    const __amdgpu_buffer_rsrc_t rw2 = MODE == SWIGLU ? buffer_rsrc(a.w2 + wbase, wbytes) : rw;
    uint32_t woff[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t r = MODE == SWIGLU ? n0 + 8 * (c >> 2) + 4 * (j & 1) + (c & 3) : n0 + 16 * (c >> 2) + 4 * j + (c & 3);
        woff[j] = (min(r, a.out - 1) - nb) * a.in + 16 * q;
    }
    // the source row of position p (any valid row past the tile's end) and where its outputs go
    auto source = [&](uint32_t p) -> uint32_t {
        const uint32_t pp = p < t.end ? p : t.m0;
        if (MODE != SWIGLU) return pp;
        return min((a.perm ? a.perm[pp] : pp) / a.kdiv, a.xrows - 1);
    };
    uint32_t to[NS];
#pragma unroll
    for (int i = 0; i < NS; i++) {
        const uint32_t p = t.m0 + 16 * i + c;
        const bool live = p < t.end;
        const uint32_t pair = a.perm ? a.perm[live ? p : t.m0] : p;
        if (MODE == SWIGLU)
            to[i] = live && pair / a.kdiv < a.xrows ? p : 0xffffffffu;
        else
            to[i] = live && pair < a.P ? pair : 0xffffffffu;
    }
    const __amdgpu_buffer_rsrc_t rx = buffer_rsrc(a.x, (uint32_t)min((uint64_t)a.xrows * a.in, (uint64_t)0xffffffffu));
    uint32_t xoff[ND], xlast[ND];  // of a step's 16 bytes, and of the last step's (past `in`: the block's first)
#pragma unroll
    for (int i = 0; i < ND; i++) {
        const uint32_t r = 8 * (kWaves * i + wv) + lane / 8, chunk = (lane % 8) ^ ((r >> 1) & 7);
        const uint32_t base = source(t.m0 + r) * a.in;
        xoff[i] = base + 16 * chunk;
        xlast[i] = tail && 16 * chunk >= tail ? base : xoff[i];
    }
    // the thread's share of the rows' scales of 16 steps: one row, kSr neighbouring steps
    constexpr int kSr = BM * kGroup / kThreads;
    const uint32_t srow = tid / (kGroup / kSr), sk = tid % (kGroup / kSr) * kSr;
    const uint16_t *sxp = a.xs + (uint64_t)source(t.m0 + srow) * nk;
    const uint32_t ob = (a.out + 127) / 128;
    const bool has_sw = tid < 2 * kGroup;
    const uint32_t swb = MODE == SWIGLU ? t.ct : min(2 * t.ct + tid / kGroup, ob - 1);
    const void *swp = MODE == SWIGLU && tid >= kGroup ? a.ws2 : a.ws;
    const uint64_t swrow = ((uint64_t)t.e * ob + swb) * nk;
    uint16_t sr[kSr];
    float swr = 0.f;
    auto load_scales = [&](uint32_t k0) {
#pragma unroll
        for (int i = 0; i < kSr; i++) sr[i] = sxp[min(k0 + sk + i, nk - 1)];
        if (has_sw) swr = scale_at(swp, a.stype, swrow + min(k0 + tid % kGroup, nk - 1));
    };
    auto keep_scales = [&](uint32_t buf) {
#pragma unroll
        for (int i = 0; i < kSr; i++) lds.sx[buf][sk + i][srow] = bf16_to_f32(sr[i]);
        if (has_sw) lds.sw[buf][tid / kGroup][tid % kGroup] = swr;
    };
    auto dma = [&](uint32_t buf, uint32_t kb) {
#pragma unroll
        for (int i = 0; i < ND; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_ptr)(lds.x[buf] + 8 * (kWaves * i + wv) * 128), 16,
                                                     kb + 1 == nk ? xlast[i] : xoff[i], kb * 128, 0, 0);
    };
    auto load_w = [&](Codes (&w)[4], uint32_t kb) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const __amdgpu_buffer_rsrc_t r = MODE == SWIGLU && j >= 2 ? rw2 : rw;
            w[j].lo = __builtin_bit_cast(u32x4q, __builtin_amdgcn_raw_buffer_load_b128(r, woff[j], kb * 128, 0));
            w[j].hi = __builtin_bit_cast(u32x4q, __builtin_amdgcn_raw_buffer_load_b128(r, woff[j] + 64, kb * 128, 0));
        }
    };
    f32x4q acc[4][NS] = {};
    Codes w[4], wn[4];
    load_scales(0);
    dma(0, 0);
    load_w(w, 0);
    for (uint32_t kb = 0; kb < nk; kb++) {
        const uint32_t buf = kb & 1, grp = kb / kGroup & 1;
        if (kb % kGroup == 0) keep_scales(grp);
        __builtin_amdgcn_s_waitcnt(0);  // this step's DMA, codes and scales are here
        __syncthreads();                // everyone's; and everyone is done with the other buffers
        if (kb + 1 < nk) {
            if ((kb + 1) % kGroup == 0) load_scales(kb + 1);
            dma(buf ^ 1, kb + 1);
            load_w(wn, kb + 1);
        }
        if (tail && kb + 1 == nk) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (16 * q >= tail) w[j].lo = u32x4q{0, 0, 0, 0};
                if (16 * q + 64 >= tail) w[j].hi = u32x4q{0, 0, 0, 0};
            }
        }
        const Operand<kF16> wo[4] = {Operand<kF16>(w[0]), Operand<kF16>(w[1]), Operand<kF16>(w[2]), Operand<kF16>(w[3])};
        const uint32_t wsel = MODE == SWIGLU ? 0 : wv >> 1;
        const float sw = lds.sw[grp][wsel][kb % kGroup];
        const float sw2 = MODE == SWIGLU ? lds.sw[grp][1][kb % kGroup] : sw;
#pragma unroll
        for (int i = 0; i < NS; i++) {
            const uint32_t r = 16 * i + c, sz = (r >> 1) & 7;
            Codes xc;
            xc.lo = *reinterpret_cast<const u32x4q *>(&lds.x[buf][r * 128 + ((q ^ sz) << 4)]);
            xc.hi = *reinterpret_cast<const u32x4q *>(&lds.x[buf][r * 128 + (((q + 4) ^ sz) << 4)]);
            const float sx = lds.sx[grp][kb % kGroup][r];
            const Operand<kF16> xo(xc);
            const float s1 = sx * sw, s2 = MODE == SWIGLU ? sx * sw2 : s1;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const f32x4q d = block_dot(wo[j], xo);
                const float s = j >= 2 ? s2 : s1;
#pragma unroll
                for (int e = 0; e < 4; e++) acc[j][i][e] = fmaf(d[e], s, acc[j][i][e]);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = wn[j];
    }
    store_tile<MODE, NS, TT>(a, acc, to, n0, t.ct, wv, lds.tops);
}

template <int MODE, int TT>
__global__ __launch_bounds__(kThreads, 2) void tile_kernel(Args a) {
    __shared__ __attribute__((aligned(16))) TileLds<16 * TT> lds;
    Tile t;
    if (!find_tile<16 * TT>(a, t, lds.find)) return;
    // token tiles in use, in steps of a quarter (32 rows of 128)
    const uint32_t live = t.end - t.m0;
    if constexpr (TT == 8) {
        if (live > 96) tile_body<MODE, TT, 8>(a, t, lds);
        else if (live > 64) tile_body<MODE, TT, 6>(a, t, lds);
        else if (live > 32) tile_body<MODE, TT, 4>(a, t, lds);
        else tile_body<MODE, TT, 2>(a, t, lds);
    } else {
        if (live > 32) tile_body<MODE, TT, 4>(a, t, lds);
        else tile_body<MODE, TT, 2>(a, t, lds);
    }
}

}  // namespace q8

static hipError_t launch_q8(Prof *p, hipStream_t s, const char *name, int mode, q8::Args a) {
    const uint32_t per_block = mode == q8::SWIGLU ? q8::kBlockRows / 2 : q8::kBlockRows;
    a.col_tiles = (a.out + per_block - 1) / per_block;
    a.kb = (a.in + 127) / 128;
    const uint32_t experts = a.offsets ? a.experts : 1;
    // DMA offsets are 32-bit
    const bool tiled = a.P > 16ull * experts && (uint64_t)a.xrows * a.in < 0xffffffffull;
    const uint32_t bm = !tiled ? 16 : mode == q8::F32OUT ? 64 : 128;
    // every non-empty segment may end in a partial tile
    const uint64_t tiles = a.P / bm + (a.offsets ? (experts < a.P ? experts : a.P) : (a.P % bm != 0));
    const uint64_t blocks = (tiles * a.col_tiles + q8::kXcds - 1) / q8::kXcds * q8::kXcds;
    if (blocks > 0x7fffffffull) return hipErrorInvalidConfiguration;
    using namespace q8;
    auto kern = tiled ? (mode == SWIGLU   ? tile_kernel<SWIGLU, 8>
                         : mode == F32OUT ? tile_kernel<F32OUT, 4>
                                          : tile_kernel<BF16OUT, 8>)
                      : (mode == SWIGLU   ? mm_kernel<SWIGLU, 1>
                         : mode == F32OUT ? mm_kernel<F32OUT, 1>
                                          : mm_kernel<BF16OUT, 1>);
    return launch_kernel(p, name, kern, dim3((uint32_t)blocks), dim3(kThreads), 0, s, a);
}

hipError_t launch_q8_rows(Prof *p, hipStream_t s, const char *name, const Q8Weight &w, const Q8Rows &x,
                          const uint32_t *offsets, const uint32_t *perm, void *y, bool bf16) {
    q8::Args a{};
    a.w = w.codes, a.ws = w.scales, a.stype = w.stype, a.in = w.in, a.out = w.out, a.experts = w.experts;
    a.x = x.codes, a.xs = x.scales, a.xrows = x.rows, a.P = x.rows;
    a.offsets = offsets, a.perm = perm, a.y = y, a.kdiv = 1;
    return launch_q8(p, s, name, bf16 ? q8::BF16OUT : q8::F32OUT, a);
}

hipError_t launch_q8_swiglu(Prof *p, hipStream_t s, const Q8Weight &gate, const Q8Weight &up, const Q8Rows &x,
                            const uint32_t *offsets, const uint32_t *perm, uint32_t k, const Q8Rows &out) {
    q8::Args a{};
    a.w = gate.codes, a.ws = gate.scales, a.w2 = up.codes, a.ws2 = up.scales, a.stype = gate.stype;
    a.in = gate.in, a.out = gate.out, a.experts = gate.experts;
    a.x = x.codes, a.xs = x.scales, a.xrows = x.rows, a.P = out.rows;
    a.offsets = offsets, a.perm = perm, a.kdiv = k;
    a.codes = out.codes, a.scales = out.scales;
    return launch_q8(p, s, "expert_swiglu_q8", q8::SWIGLU, a);
}

}  // namespace moehip
