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
#include <type_traits>

#include "q8.hpp"

namespace moehip {

namespace q8 {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

enum { SWIGLU = 0, F32OUT = 1, BF16OUT = 2, ACT = 3 };  // ACT: SwiGLU as F32 rows

struct Args {
    const uint8_t *w, *w2;        // codes (w2: the up weights of SWIGLU)
    const void *ws, *ws2;         // block scales, of type `stype`
    const uint8_t *x;             // input rows' codes [xrows, in]
    const uint16_t *xs;           // and scales [xrows, kb]
    const uint32_t *offsets;      // [experts + 1], or null: one segment of all positions
    const uint32_t *perm;         // [P] pair of each position, or null: the position itself
    void *y;                      // F32OUT / BF16OUT / ACT: [P, out]
    uint32_t *list;               // ACT: the number of tiles, one word unused, first position and end of each
    uint8_t *codes;               // SWIGLU: [P, out] and scales [P, ceil(out / 128)]
    uint16_t *scales;
    uint32_t stype, xrows, in, out, kb, experts, P, kdiv;
    uint32_t col_tiles;           // tiles along the outputs
    uint32_t tiles;               // at most this many along the positions
};

// The work of a block: items, each an M-tile (a run of at most BM positions of a
// segment, experts ascending) times a column tile.  Workgroup b runs on XCD
// b % 8; the items are split into eight contiguous ranges, one per XCD, so the
// tiles that share an expert's weights and a run's rows meet in one L2; the
// blocks of an XCD take its range's items in turn.  Segments of many tiles both
// ways go by panels of kPanel column tiles, so that the 32 items an XCD has in
// hand read 4 tiles of weights and 8 of tokens rather than all weights (4096 rows,
// 4096 to 12288 columns: 200 us; 205 with panels of 8, 224 of 1, 247 of all).
// Every thread of the block calls it; slots `from` and on of the block are written to out[0 .. n), at most
// kMax; n is returned.  Offsets past P count as P and a segment that ends before
// it starts is empty.  `list`: where the launch leaves its tiles, for the next one.
struct Tile {
    uint32_t e, m0, end, ct;
};
constexpr uint32_t kXcds = 8, kPanel = 4;
template <int BM, int NW>
__device__ __forceinline__ uint32_t find_items(const Args &a, uint32_t from, uint32_t kMax, Tile *out, uint32_t *lds /* NW */,
                                               uint32_t *list = nullptr) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const uint32_t per = (a.experts + 64 * NW - 1) / (64 * NW), e0 = tid * per;
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
            mine = min(mine + n, a.tiles);
        }
        uint32_t incl = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(incl, d);
            if ((int)lane >= d) incl = __builtin_elementwise_add_sat(incl, up);
        }
        if (lane == 63) lds[wv] = incl;
        __syncthreads();
        before = incl - mine;
        total = 0;
#pragma unroll
        for (uint32_t v = 0; v < NW; v++) {
            if (v < wv) before = __builtin_elementwise_add_sat(before, lds[v]);
            total = __builtin_elementwise_add_sat(total, lds[v]);
        }
    }
    // (fewer than 2^31 items: the launch checks it.  Segments that overlap can make
    // more tiles than the launch has blocks for, and than 32 bits count: sums stop at
    // 2^32 - 1 and a thread's tiles at a.tiles, the last tiles are left out.)
    total = min(total, a.tiles);
    if (list && blockIdx.x == 0 && tid == 0) list[0] = total;
    const uint32_t items = total * a.col_tiles, range = (items + kXcds - 1) / kXcds;
    const uint32_t lo_item = blockIdx.x % kXcds * range, hi_item = min(items, lo_item + range);
    const uint32_t turn = gridDim.x / kXcds;
    const uint32_t first = lo_item + blockIdx.x / kXcds + from * turn;
    if (first >= hi_item) return 0;
    const uint32_t n = min(kMax, (hi_item - first + turn - 1) / turn);
    // item `i` of a segment of k tiles, none of which `total` cuts off: a tile gets all of
    // its columns or none
    auto put = [&](uint32_t s, uint32_t e, uint32_t lo, uint32_t hi, uint32_t k, uint32_t first_tile, uint32_t i) {
        const uint32_t panel = k < 2 * kPanel || a.col_tiles <= 2 * kPanel ? a.col_tiles : kPanel;
        const uint32_t ct = i / (k * panel) * panel;
        const uint32_t wide = min(panel, a.col_tiles - ct), at = i - k * ct;
        const uint32_t m0 = lo + at / wide * BM, end = hi - m0 < BM ? hi : m0 + BM;
        out[s] = Tile{e, m0, end, ct + at % wide};
        if (list && ct + at % wide == 0) {
            uint32_t *const l = list + 2 + 2 * (first_tile + at / wide);
            l[0] = m0, l[1] = end;
        }
    };
    if (!a.offsets) {
        if (tid < n) put(tid, 0, 0, a.P, total, 0, first + tid * turn);
    } else {
        for (uint32_t s = 0; s < n; s++) {
            const uint32_t item = first + s * turn, tile = item / a.col_tiles;
            if (tile < before || tile >= before + mine) continue;
            uint32_t at = before;
            for (uint32_t i = 0; i < per && e0 + i < a.experts; i++) {
                uint32_t lo, k;
                const uint32_t hi = seg(e0 + i, lo, k);
                if (tile - at < k) {
                    put(s, e0 + i, lo, hi, min(k, total - at), at, item - at * a.col_tiles);
                    break;
                }
                at += k;
            }
        }
    }
    __syncthreads();
    return n;
}
// The one item of a block in a grid with a block per item.
constexpr int kFind = 12;  // its words of LDS
template <int BM, int NW>
__device__ __forceinline__ bool find_tile(const Args &a, Tile &t, uint32_t *lds, uint32_t *list) {
    static_assert(NW + 4 <= kFind, "LDS words");
    Tile *out = reinterpret_cast<Tile *>(lds + NW);
    if (find_items<BM, NW>(a, 0, 1, out, lds, list) == 0) return false;
    t.e = __builtin_amdgcn_readfirstlane(out->e);
    t.m0 = __builtin_amdgcn_readfirstlane(out->m0);
    t.end = __builtin_amdgcn_readfirstlane(out->end);
    t.ct = __builtin_amdgcn_readfirstlane(out->ct);
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

// The outputs of a wave's row tiles for NS token tiles of 16: acc[j][i] holds row
// tile j, token tile i; the lane's rows are neighbours from `col` on; to[i] is
// where the lane's token of tile i goes.
typedef __bf16 bf16x2q __attribute__((ext_vector_type(2)));
typedef float f32x2q __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {  // nearest even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2q{a, b}, bf16x2q));
}
template <int MODE, int RT, int NS>
__device__ __forceinline__ void store_rows(const Args &a, const f32x4q (&acc)[RT][NS], const uint32_t (&to)[NS],
                                           uint32_t col) {
    // 16-byte stores of whole groups (4 F32, 8 bf16) where every row starts aligned
    constexpr int G = MODE == BF16OUT && RT > 1 ? 8 : 4;
    const bool vec = a.out % G == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15u) == 0;
#pragma unroll
    for (int i = 0; i < NS; i++) {
        if (to[i] == 0xffffffffu) continue;
        const uint64_t at = (uint64_t)to[i] * a.out + col;
        if constexpr (MODE == F32OUT) {
            float *y = static_cast<float *>(a.y) + at;
#pragma unroll
            for (int j = 0; j < RT; j++) {
                if (vec) {
                    if (col + 4 * j < a.out) *reinterpret_cast<f32x4q *>(y + 4 * j) = acc[j][i];
                } else {
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (col + 4 * j + r < a.out) y[4 * j + r] = acc[j][i][r];
                }
            }
        } else {
            uint16_t *y = static_cast<uint16_t *>(a.y) + at;
            uint32_t b[2 * RT];
#pragma unroll
            for (int j = 0; j < RT; j++) {
                b[2 * j] = bf16_pair(acc[j][i][0], acc[j][i][1]);
                b[2 * j + 1] = bf16_pair(acc[j][i][2], acc[j][i][3]);
            }
            if (vec) {
                if constexpr (G == 8) {
#pragma unroll
                    for (int j = 0; j < RT; j += 2)
                        if (col + 4 * j < a.out)
                            *reinterpret_cast<u32x4q *>(y + 4 * j) = u32x4q{b[2 * j], b[2 * j + 1], b[2 * j + 2], b[2 * j + 3]};
                } else {
                    if (col < a.out) *reinterpret_cast<u32x2q *>(y) = u32x2q{b[0], b[1]};
                }
            } else {
#pragma unroll
                for (int r = 0; r < 4 * RT; r++)
                    if (col + r < a.out) y[r] = (uint16_t)(b[r / 2] >> (16 * (r % 2)));
            }
        }
    }
}

// silu(g) * u.  The rounding of log2(e) * g puts the exponential off by up to
// |g| 2^-23 of it: 2^-16 where silu(g) is not yet 0, far below the 2^-4 of the 8-bit
// codes this becomes.
__device__ __forceinline__ float swiglu_of(float g, float u) {
    constexpr float kLog2e = 1.44269504f;
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * g)) * u;
}

// SWIGLU: row tiles 0 .. RT/2 - 1 of acc are gate rows, the rest their up rows.
// The waves of the block hold 128 output columns of its tokens: the largest
// magnitude of each token goes through LDS (tops: [NW][16 NS]).
template <int RT, int NS, int NW>
__device__ __forceinline__ void store_swiglu(const Args &a, const f32x4q (&acc)[RT][NS], const uint32_t (&to)[NS],
                                             uint32_t col, uint32_t ct, uint32_t wv, uint32_t *tops) {
    constexpr int V = 2 * RT, BM = 16 * NS;  // V: columns a lane holds
    const uint32_t lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4, ob = (a.out + 127) / 128;
    const bool cols_in = col < a.out;  // (out is a multiple of 16: all of the lane's columns or none)
    float act[NS][V];
#pragma unroll
    for (int i = 0; i < NS; i++) {
        uint32_t top = 0;
#pragma unroll
        for (int r = 0; r < V; r++) {
            const float g = acc[r / 4][i][r % 4], u = acc[RT / 2 + r / 4][i][r % 4];
            act[i][r] = swiglu_of(g, u);
            if (cols_in) top = max(top, abs_word(act[i][r]));
        }
        top = max_xor32_u(max_xor16_u(top));
        if (q == 0) tops[wv * BM + 16 * i + c] = top;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NS; i++) {
        const uint32_t at = 16 * i + c;
        uint32_t top = tops[at];
#pragma unroll
        for (int v = 1; v < NW; v++) top = max(top, tops[v * BM + at]);
        const uint32_t sb = q8_scale_bits(top);
        if (to[i] == 0xffffffffu) continue;
        const float r = q8_inverse(sb);
        if (cols_in) {
            uint32_t *o = reinterpret_cast<uint32_t *>(a.codes + (uint64_t)to[i] * a.out + col);
            if constexpr (V == 8)
                *reinterpret_cast<u32x2q *>(o) =
                    u32x2q{q8_codes4(act[i][0], act[i][1], act[i][2], act[i][3], r),
                           q8_codes4(act[i][4], act[i][5], act[i][6], act[i][7], r)};
            else
                *o = q8_codes4(act[i][0], act[i][1], act[i][2], act[i][3], r);
        }
        if (wv == 0 && q == 0) a.scales[(uint64_t)to[i] * ob + ct] = (uint16_t)sb;
    }
}

// Few rows per expert: the time is the weights' way from memory, so what counts
// is how many of their loads are in flight.  A wave owns RT row tiles (SWIGLU: 16
// gate rows and their up rows) and a range of the blocks of 128 columns (KS waves
// share rows; their sums join through LDS in order); the codes of D blocks are
// loaded ahead into registers, the token rows' with them.  The scales of up to
// kChunk blocks wait in LDS as F32, loaded before the codes so that their wait
// leaves the codes in flight.
//
// Bound by the weights' bytes once there are a few MiB of them: 128 rows over
// 128 experts, 768 columns to 2048, bf16, 24.3 us or 5.4 TB/s; 1280 rows over 512
// experts of 512 columns, 97.9 us or 5.1 TB/s; one row, 2048 columns to 65536,
// 21.4 us or 6.3 TB/s, the rate of a read.  Below, by the launch and one pass of
// loads: one row, 2048 columns to 4096, 4.2 us, of which an empty launch is 4 (18
// with one block ahead and no split of the columns).  Where there are rows enough,
// two blocks ahead in 16 waves a CU beat four in 8 (192 rows over 128 experts, 768
// columns to 2048, F32: 34 us, 40).
constexpr uint32_t kChunk = 64;

template <int MODE, int RT, int TT, int KS, int NW>
struct StreamLds {
    float sx[kChunk][16 * TT];
    float sw[MODE == SWIGLU || MODE == ACT ? 2 : 1][kChunk];
    float red[KS > 1 ? NW - NW / KS : 1][KS > 1 ? 64 * RT * TT * 4 : 1];
    uint32_t tops[MODE == SWIGLU ? NW * 16 * TT : 1];
    uint32_t find[kFind];
};

template <int MODE, int RT, int TT, int KS, int NW, int D, int WPS>
__global__ __launch_bounds__(64 * NW, WPS) void stream_kernel(Args a) {
    constexpr bool kF16 = MODE == F32OUT, kGated = MODE == SWIGLU || MODE == ACT;
    constexpr int BM = 16 * TT, RG = NW / KS;  // RG: groups of rows in the block
    constexpr int kCols = kGated ? 16 : 16 * RT;  // outputs of a wave
    static_assert(!kGated || RT == 2, "gate rows and their up rows");
    static_assert(MODE != SWIGLU || (KS == 1 && NW == 8), "128 output columns a block");
    static_assert(RG * kCols <= 128 && 128 % (RG * kCols) == 0, "a block's rows share their scales");
    __shared__ __attribute__((aligned(16))) StreamLds<MODE, RT, TT, KS, NW> lds;
    Tile t;
    if (!find_tile<BM, NW>(a, t, lds.find, MODE == ACT ? a.list : nullptr)) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63, c = lane & 15, q = lane >> 4;
    const uint32_t wv = __builtin_amdgcn_readfirstlane(tid >> 6), rg = wv / KS, ks = wv % KS;
    const uint32_t n0 = t.ct * (RG * kCols) + rg * kCols, nb = min(n0, a.out - 1);
    const uint32_t nk = a.kb, tail = a.in % 128, ob = (a.out + 127) / 128;
    // weights: one resource per matrix from row nb on, a lane's rows as offsets
    // (rows past `out` repeat the last and are not stored)
    const uint64_t wbase = ((uint64_t)t.e * a.out + nb) * a.in;
    const uint32_t wbytes = (uint32_t)min((uint64_t)(a.out - nb) * a.in, (uint64_t)0xffffffffu);
    const __amdgpu_buffer_rsrc_t rw = buffer_rsrc(a.w + wbase, wbytes);
    const __amdgpu_buffer_rsrc_t rw2 = kGated ? buffer_rsrc(a.w2 + wbase, wbytes) : rw;
    uint32_t woff[RT];
#pragma unroll
    for (int j = 0; j < RT; j++) {
        const uint32_t r = kGated ? n0 + c : n0 + 4 * RT * (c >> 2) + 4 * j + (c & 3);
        woff[j] = (min(r, a.out - 1) - nb) * a.in;
    }
    // positions past the tile's end read its first row; outputs go to to[]
    auto source = [&](uint32_t p) -> uint32_t {
        const uint32_t pp = p < t.end ? p : t.m0;
        if (!kGated) return pp;
        return min((a.perm ? a.perm[pp] : pp) / a.kdiv, a.xrows - 1);
    };
    const uint8_t *xrow[TT];
    uint32_t to[TT];
#pragma unroll
    for (int i = 0; i < TT; i++) {
        const uint32_t p = t.m0 + 16 * i + c;
        const bool live = p < t.end;
        const uint32_t pair = a.perm ? a.perm[live ? p : t.m0] : p;
        if (kGated)
            to[i] = live && pair / a.kdiv < a.xrows ? p : 0xffffffffu;
        else
            to[i] = live && pair < a.P ? pair : 0xffffffffu;
        xrow[i] = a.x + (uint64_t)source(p) * a.in;
    }
    const uint64_t swrow = ((uint64_t)t.e * ob + min(n0 / 128, ob - 1)) * nk;
    f32x4q acc[RT][TT] = {};
    for (uint32_t k0 = 0; k0 < nk; k0 += kChunk) {
        const uint32_t kn = min(kChunk, nk - k0);        // blocks of this chunk
        const uint32_t len = (kn + KS - 1) / KS;         // and of the wave's range in it
        const uint32_t kbeg = ks * len, kend = min(kbeg + len, kn);
        if (k0) __syncthreads();                         // the last chunk's scales are read
        for (uint32_t i = tid; i < kn * BM; i += 64 * NW)
            lds.sx[i / BM][i % BM] = bf16_to_f32(a.xs[(uint64_t)source(t.m0 + i % BM) * nk + k0 + i / BM]);
        if (tid < kn) {
            lds.sw[0][tid] = scale_at(a.ws, a.stype, swrow + k0 + tid);
            if constexpr (kGated) lds.sw[1][tid] = scale_at(a.ws2, a.stype, swrow + k0 + tid);
        }
        Codes w[D][RT], x[D][TT];
        auto load = [&](int d, uint32_t kb) {  // blocks past the chunk's end: its last again, with a scale of zero
            const uint32_t k = k0 + min(kb, kn - 1), k128 = k * 128;
            const bool last = tail && k + 1 == nk;  // chunks past `in` read the block's first
            const uint32_t lo = last && 16 * q >= tail ? 0 : 16 * q, hi = last && 16 * q + 64 >= tail ? 0 : 16 * q + 64;
#pragma unroll
            for (int j = 0; j < RT; j++) {
                const __amdgpu_buffer_rsrc_t r = kGated && j == 1 ? rw2 : rw;
                w[d][j].lo = __builtin_bit_cast(u32x4q, __builtin_amdgcn_raw_buffer_load_b128(r, woff[j] + lo, k128, 0));
                w[d][j].hi = __builtin_bit_cast(u32x4q, __builtin_amdgcn_raw_buffer_load_b128(r, woff[j] + hi, k128, 0));
            }
#pragma unroll
            for (int i = 0; i < TT; i++) {
                const uint8_t *row = xrow[i] + k128;
                x[d][i].lo = *reinterpret_cast<const u32x4q *>(row + lo);
                x[d][i].hi = *reinterpret_cast<const u32x4q *>(row + hi);
            }
        };
        auto use = [&](int d, uint32_t kb) {
            const uint32_t kc = min(kb, kn - 1);
            const bool live = kb < kend;
            if (tail && k0 + kc + 1 == nk) {
#pragma unroll
                for (int j = 0; j < RT; j++) {
                    if (16 * q >= tail) w[d][j].lo = u32x4q{0, 0, 0, 0};
                    if (16 * q + 64 >= tail) w[d][j].hi = u32x4q{0, 0, 0, 0};
                }
            }
            const float sw = live ? lds.sw[0][kc] : 0.f;
            const float sw2 = kGated ? (live ? lds.sw[kGated][kc] : 0.f) : sw;
#pragma unroll
            for (int i = 0; i < TT; i++) {
                const Operand<kF16> xo(x[d][i]);
                const float sx = live ? lds.sx[kc][16 * i + c] : 0.f;
#pragma unroll
                for (int j = 0; j < RT; j++) {
                    const f32x4q p = block_dot(Operand<kF16>(w[d][j]), xo);
                    const float s = sx * (kGated && j == 1 ? sw2 : sw);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[j][i][e] = fmaf(p[e], s, acc[j][i][e]);
                }
            }
        };
#pragma unroll
        for (int d = 0; d < D; d++) load(d, kbeg + d);
        __syncthreads();
        uint32_t kb = kbeg;
        for (; kb + D < kend; kb += D) {
#pragma unroll
            for (int d = 0; d < D; d++) {
                use(d, kb + d);
                load(d, kb + D + d);
            }
        }
#pragma unroll
        for (int d = 0; d < D; d++) use(d, kb + d);
    }
    if constexpr (KS > 1) {
        if (ks > 0) {
            float *r = lds.red[rg * (KS - 1) + ks - 1];
#pragma unroll
            for (int j = 0; j < RT; j++)
#pragma unroll
                for (int i = 0; i < TT; i++)
                    *reinterpret_cast<f32x4q *>(r + ((j * TT + i) * 64 + lane) * 4) = acc[j][i];
        }
        __syncthreads();
        if (ks > 0) return;
#pragma unroll
        for (int v = 0; v < KS - 1; v++)
#pragma unroll
            for (int j = 0; j < RT; j++)
#pragma unroll
                for (int i = 0; i < TT; i++)
                    acc[j][i] += *reinterpret_cast<const f32x4q *>(lds.red[rg * (KS - 1) + v] + ((j * TT + i) * 64 + lane) * 4);
    }
    if constexpr (MODE == SWIGLU)
        store_swiglu<RT, TT, NW>(a, acc, to, n0 + 4 * q, t.ct, wv, lds.tops);
    else if constexpr (MODE == ACT) {
        if (n0 + 4 * q >= a.out) return;  // (out is a multiple of 16)
#pragma unroll
        for (int i = 0; i < TT; i++) {
            if (to[i] == 0xffffffffu) continue;
            f32x4q v;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = swiglu_of(acc[0][i][e], acc[1][i][e]);
            *reinterpret_cast<f32x4q *>(static_cast<float *>(a.y) + (uint64_t)to[i] * a.out + n0 + 4 * q) = v;
        }
    } else
        store_rows<MODE, RT, TT>(a, acc, to, n0 + 4 * RT * q);
}

// The same product for many rows per expert: items of 128 tokens and 256 weight
// rows (SWIGLU: 128 gate rows and their up rows) for blocks of eight waves, one
// a CU, that take one item after another.  A step is a block of 128 columns: its
// token and weight rows reach LDS by buffer DMA (eight rows of 128 bytes an
// instruction, so that neighbouring lanes read neighbouring bytes: loads in
// the matrix cores' own layout, 16 rows an instruction, took four times as long),
// two steps ahead and across the items' borders; 16-byte chunks are XOR-swizzled
// by half the row number, so that 16 rows' equal chunks lie in distinct banks.
// The waves form 4 x 2: 64 weight rows times 64 tokens (every other tile of 16)
// each, so that LDS is read 2 x 64 rows of 128 bytes for 16 matrix instructions.
// One barrier a step.  The rows an item reads and writes are looked up once for
// kSlots items.
//
// 4096 rows, 4096 columns to 12288, bf16: 200 us, 2060 TFLOP/s; 4001 rows, 2048 to
// 4096: 39.6 us, 1695.  A step takes 1750 cycles: 1024 of matrix instructions; 768 of
// DMA at the 64 bytes a cycle a CU loads, which hold up the waves that issue them;
// the scaling (64 FMA a wave) and reads of LDS fill the rest.  An item's first
// loads and its outputs come to another 3500 cycles, the launch's to 7000.
// (The second product on the way here, before panels: 47.2 us with a step's DMA in
// one go, 45.0 between the products, 43 with the operands read a step ahead, 41
// with whole lines out.  Waves that issue the DMA at different points, by branches:
// 42.6 to 52.9 where all at once took 40.4; wave priorities: no difference.)
typedef __attribute__((address_space(3))) void *lds_ptr;
constexpr uint64_t kCus = 256;
constexpr uint32_t kStage = 128 * 128;  // bytes of a stage's token rows, half of its weight rows'
constexpr int kScaleSlots = 32, kGroup = 8, kStages = 3, kTileWaves = 8, kTileRows = 128, kSlots = 8;

struct TileLds {
    uint8_t x[kStages * kStage];
    uint8_t w[2 * kStages * kStage];
    uint16_t sx[kScaleSlots][kTileRows];  // scales by step, in a ring of four groups of kGroup steps
    float sw[kScaleSlots][2];
    uint32_t tops[4 * kTileRows];
    uint32_t map[kSlots][kTileRows];  // SWIGLU: input row of each position; else its output row; 0xffffffff: none
    Tile slot[kSlots];
    uint32_t scan[kTileWaves];
};

// TAIL: `in` is no multiple of 128
template <int MODE, bool TAIL>
__global__ __launch_bounds__(64 * kTileWaves, 2) void tile_kernel(Args a) {
    constexpr bool kF16 = MODE == F32OUT;
    constexpr int NX = 2, NW = 4;     // DMA instructions of a wave and step: token rows, weight rows
    constexpr int kLoads = NX + NW;
    __shared__ __attribute__((aligned(16))) TileLds lds;
    const uint32_t tid = threadIdx.x, lane = tid & 63, c = lane & 15, q = lane >> 4;
    const uint32_t wv = __builtin_amdgcn_readfirstlane(tid >> 6), wg = wv >> 1, tg = wv & 1;
    const uint32_t nk = a.kb, tail = TAIL ? a.in % 128 : 0, ob = (a.out + 127) / 128;
    const __amdgpu_buffer_rsrc_t rx = buffer_rsrc(a.x, (uint32_t)((uint64_t)a.xrows * a.in));
    const uint32_t wbytes = (uint32_t)((uint64_t)a.out * a.in);
    // DMA: instruction i of wave wv fills LDS rows 8 (8 i + wv) .. + 7; lane l
    // writes chunk l % 8 of row l / 8.  LDS row 64 g + 16 j + c holds the row that is
    // row c of row tile j of the waves of group g: four row tiles interleave, so that a
    // lane's results are neighbouring outputs (SWIGLU: tiles 0, 1 gate, 2, 3 up).
    const uint32_t drow = 8 * wv + lane / 8;  // + 64 i
    const uint32_t dchunk = ((lane % 8) ^ ((drow >> 1) & 7)) * 16;
    const uint32_t dc = drow % 16, dj = drow / 16 % 4;
    const uint32_t dlocal = MODE == SWIGLU ? 8 * (dc >> 2) + 4 * (dj & 1) + (dc & 3) : 16 * (dc >> 2) + 4 * dj + (dc & 3);
    // the item whose steps are being loaded
    __amdgpu_buffer_rsrc_t rw = rx;
    uint32_t xoff[NX] = {}, woff[NW] = {}, sxoff = 0, swoff = 0;
    // the thread's share of the scales of kGroup steps: kSr neighbouring steps of one row
    constexpr int kSr = kTileRows * kGroup / (64 * kTileWaves);
    const uint32_t srow = tid / (kGroup / kSr), sk = tid % (kGroup / kSr) * kSr;
    const bool has_sw = tid < 2 * kGroup;
    auto aim = [&](uint32_t s) {
        const Tile t = lds.slot[s];
        const uint32_t e = __builtin_amdgcn_readfirstlane(t.e);
        const uint8_t *w = MODE == SWIGLU && wv >= 4 ? a.w2 : a.w;  // (SWIGLU: the wave's rows are all of one matrix)
        rw = buffer_rsrc(w + (uint64_t)e * a.out * a.in, wbytes);
        // rows past `out` repeat the last and are not stored
#pragma unroll
        for (int i = 0; i < NW; i++)
            woff[i] = min((MODE == SWIGLU ? t.ct * 128 + 32 * i : t.ct * 256 + 64 * i) + dlocal, a.out - 1) * a.in + dchunk;
        // positions past the item's end, and those that name no row, read some row
        auto source = [&](uint32_t r) {
            return MODE == SWIGLU ? min(lds.map[s][r], a.xrows - 1) : t.m0 + r < t.end ? t.m0 + r : t.m0;
        };
#pragma unroll
        for (int i = 0; i < NX; i++) xoff[i] = source(drow + 64 * i) * a.in + dchunk;
        sxoff = source(srow) * nk;
        swoff = (e * ob + (MODE == SWIGLU ? t.ct : min(2 * t.ct + tid / kGroup, ob - 1))) * nk;
    };
    // columns past `in` in the last step: a chunk is replaced by its row's first of
    // the block, and the weights' codes are zeroed when they are used
    const uint32_t back = TAIL && dchunk >= tail ? dchunk : 0;
    // one of the kLoads instructions of the block at column k into the stage at `to`
    // (stages are named by where their token rows start)
    auto load = [&](int i, uint32_t to, uint32_t k) {
        const uint32_t b = TAIL && k + 128 > a.in ? back : 0;
        if (i < NX)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_ptr)(lds.x + to + (64 * i + 8 * wv) * 128), 16,
                                                     xoff[i < NX ? i : 0] - b, k, 0, 0);
        else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_ptr)(lds.w + 2 * to + (64 * (i - NX) + 8 * wv) * 128), 16,
                                                     woff[i < NX ? 0 : i - NX] - b, k, 0, 0);
    };
    uint16_t sr[kSr];
    float swr = 0.f;
    auto load_scales = [&](uint32_t k0) {
#pragma unroll
        for (int i = 0; i < kSr; i++) sr[i] = a.xs[sxoff + min(k0 + sk + i, nk - 1)];
        const void *from = MODE == SWIGLU && tid >= kGroup ? a.ws2 : a.ws;
        if (has_sw) swr = scale_at(from, a.stype, swoff + min(k0 + tid % kGroup, nk - 1));
    };
    auto keep_scales = [&](uint32_t buf) {
#pragma unroll
        for (int i = 0; i < kSr; i++) lds.sx[buf + sk + i][srow] = sr[i];
        if (has_sw) lds.sw[buf + tid % kGroup][tid / kGroup] = swr;
    };
    // a lane's chunks of its row in tile 0 of a wave's rows
    const uint32_t lo = c * 128 + ((q ^ (c >> 1)) << 4), hi = c * 128 + (((q + 4) ^ (c >> 1)) << 4);
    const uint8_t *const xbase = lds.x + 16 * tg * 128, *const wbase = lds.w + 64 * wg * 128;
    auto codes = [&](const uint8_t *rows) {
        return Codes{*reinterpret_cast<const u32x4q *>(rows + lo), *reinterpret_cast<const u32x4q *>(rows + hi)};
    };
    auto weights = [&](uint32_t stage, int j) { return codes(wbase + 2 * stage + j * 2048); };
    auto tokens = [&](uint32_t stage, int i) { return codes(xbase + stage + i * 4096); };
    // What a wave holds of a step: its scales, raw, and its codes of NS token tiles
    // (tile i: rows 32 i + 16 tg on) and four row tiles.
    struct Scales {
        float sw, sw2;
        uint32_t sx[4];
    };
    auto scales = [&](auto &sc, uint32_t slot) {
        sc.sw = lds.sw[slot][MODE == SWIGLU ? 0 : wg >> 1];
        sc.sw2 = MODE == SWIGLU ? lds.sw[slot][1] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) sc.sx[i] = lds.sx[slot][32 * i + 16 * tg + c];
    };
    // A step over codes wc, xc and scales sc; each is replaced by the next step's
    // after its last use (from stage `next` and the scales' slot), and issue(i),
    // i <= kLoads, is called along the products (a step's DMA in one go held the waves
    // up until the memory pipe had taken all of it).  A block's sums join their running
    // sums kLag products later.  In this order the matrix cores wait for neither.
    auto compute = [&](auto &acc, Codes (&wc)[4], auto &xc, Scales &sc, uint32_t next, uint32_t slot, bool last,
                       auto issue) {
        constexpr int NS = sizeof(acc[0]) / sizeof(acc[0][0]), kLag = 3;
        if (TAIL && last) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (16 * q >= tail) wc[j].lo = u32x4q{0, 0, 0, 0};
                if (16 * q + 64 >= tail) wc[j].hi = u32x4q{0, 0, 0, 0};
            }
        }
        const Operand<kF16> wo[4] = {Operand<kF16>(wc[0]), Operand<kF16>(wc[1]), Operand<kF16>(wc[2]), Operand<kF16>(wc[3])};
        float s1[NS], s2[NS];
#pragma unroll
        for (int i = 0; i < NS; i++) {
            s1[i] = bf16_to_f32(sc.sx[i]) * sc.sw;
            s2[i] = MODE == SWIGLU ? bf16_to_f32(sc.sx[i]) * sc.sw2 : 0.f;
        }
        f32x4q d[4 * NS];
#pragma unroll
        for (int n = 0; n < 4 * NS + kLag; n++) {
            const int i = n / 4, j = n % 4;
            if (n < 4 * NS) {
                d[n] = block_dot(wo[j], Operand<kF16>(xc[i]));
                if (i == NS - 1) wc[j] = weights(next, j);
                if (j == 3) xc[i] = tokens(next, i);
                if (n == 1) issue(0);
                if (n == 3) scales(sc, slot);
                if (n >= 3) {
                    constexpr int R = 4 * NS - 3;
#pragma unroll
                    for (int l = (n - 3) * kLoads / R; l < (n - 2) * kLoads / R; l++) issue(l + 1);
                }
            }
            if (n >= kLag) {
                const int m = n - kLag;
                const float s = MODE == SWIGLU && m % 4 >= 2 ? s2[m / 4] : s1[m / 4];
#pragma unroll
                for (int e = 0; e < 4; e++) acc[m % 4][m / 4][e] = fmaf(d[m][e], s, acc[m % 4][m / 4][e]);
            }
            if constexpr (!kF16) __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (uint32_t from = 0;; from += kSlots) {
        const uint32_t slots = find_items<kTileRows, kTileWaves>(a, from, kSlots, lds.slot, lds.scan);
        if (slots == 0) return;
        for (uint32_t i = tid; i < slots * kTileRows; i += 64 * kTileWaves) {
            const Tile t = lds.slot[i / kTileRows];
            const uint32_t p = t.m0 + i % kTileRows;
            uint32_t to = 0xffffffffu;
            if (p < t.end) {
                to = a.perm ? a.perm[p] : p;
                if constexpr (MODE == SWIGLU) to /= a.kdiv;
                if (to >= (MODE == SWIGLU ? a.xrows : a.P)) to = 0xffffffffu;
            }
            lds.map[i / kTileRows][i % kTileRows] = to;
        }
        __syncthreads();
        // the step that is loaded next: slot ps (past the last: the last again,
        // unused), column pk; whether it begins a group of scales; the group's ring slot
        uint32_t ps = 0, pk = 0, pslot = kScaleSlots - kGroup;
        bool due = true, pending = false;
        const uint32_t columns = nk * 128;
        // part i of its loads, in order 0 .. kLoads: its scales come first, so that the
        // wait for it covers them
        auto load_part = [&](int i, uint32_t to) {
            if (i == 0) {
                if (due) {
                    if (pk == 0) aim(min(ps, slots - 1));
                    load_scales(pk / 128);
                    pslot = (pslot + kGroup) % kScaleSlots;
                }
                pending = due;
                __builtin_amdgcn_sched_barrier(0);
            } else {
                load(i - 1, to, pk);
            }
            if (i < kLoads) return;
            pk += 128;
            if (pk == columns) pk = 0, ps++;
            due = pk % (kGroup * 128) == 0;
        };
        auto ahead = [&](uint32_t to) {
#pragma unroll
            for (int i = 0; i <= kLoads; i++) load_part(i, to);
        };
        auto barrier = [&] {  // of LDS traffic only: the loads stay in flight
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4) | (0 << 8));
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        auto store_scales = [&] {
            if (pending) keep_scales(pslot);
        };
        // A step begins when the next one's rows are in LDS and this one's are read
        // out: all but the loads of the step after the next have landed (gfx9
        // encoding: vmcnt), everyone's.  Before an item's outputs all of them have
        // (`landed`), so that its next step does not wait for the stores.
        bool landed = false;
        auto begin = [&] {
            __builtin_amdgcn_sched_barrier(0);
            if (!landed) __builtin_amdgcn_s_waitcnt(kLoads | (7 << 4) | (15 << 8));
            landed = false;
            store_scales();
            barrier();
        };
        ahead(0);
        store_scales();
        ahead(kStage);
        begin();
        ahead(2 * kStage);
        // the stages of the step at work and of the next one; the ring slot of the
        // item's first scales
        uint32_t cur = 0, next = kStage, slot0 = 0;
        // An item's outputs, through the stage `buf`: a lane's results are neighbours
        // of one row, but neighbouring lanes hold different rows, and stores of that
        // kind took 64 times a line each.  16-byte chunks are XOR-swizzled by their row.
        auto outputs = [&](auto &acc, uint32_t s, uint32_t buf) {
            constexpr int NS = sizeof(acc[0]) / sizeof(acc[0][0]);
            const Tile t = lds.slot[s];
            const uint32_t ct = __builtin_amdgcn_readfirstlane(t.ct);
            if constexpr (MODE == SWIGLU) {
                float act[NS][8];
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    uint32_t top = 0;
#pragma unroll
                    for (int r = 0; r < 8; r++) {
                        act[i][r] = swiglu_of(acc[r / 4][i][r % 4], acc[2 + r / 4][i][r % 4]);
                        top = max(top, abs_word(act[i][r]));
                    }
                    // (out is a multiple of 16: all of the lane's columns count, or none)
                    if (ct * 128 + wg * 32 + 8 * q >= a.out) top = 0;
                    top = max_xor32_u(max_xor16_u(top));
                    if (q == 0) lds.tops[wg * kTileRows + 32 * i + 16 * tg + c] = top;
                }
                barrier();
                auto scale_of = [&](uint32_t row) {
                    const uint32_t *p = lds.tops + row;
                    return q8_scale_bits(max(max(p[0], p[kTileRows]), max(p[2 * kTileRows], p[3 * kTileRows])));
                };
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    const uint32_t row = 32 * i + 16 * tg + c, chunk = 2 * wg + (q >> 1);
                    const float r = q8_inverse(scale_of(row));
                    *reinterpret_cast<u32x2q *>(lds.x + buf + row * 128 + ((chunk ^ (row & 7)) << 4) + 8 * (q & 1)) =
                        u32x2q{q8_codes4(act[i][0], act[i][1], act[i][2], act[i][3], r),
                               q8_codes4(act[i][4], act[i][5], act[i][6], act[i][7], r)};
                }
                barrier();
                if (tid < t.end - t.m0 && lds.map[s][tid] != 0xffffffffu)
                    a.scales[(uint64_t)(t.m0 + tid) * ob + ct] = (uint16_t)scale_of(tid);
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    const uint32_t row = 16 * wv + 8 * m + lane / 8, chunk = lane % 8, col = ct * 128 + 16 * chunk;
                    if (row < t.end - t.m0 && lds.map[s][row] != 0xffffffffu && col < a.out)
                        *reinterpret_cast<u32x4q *>(a.codes + (uint64_t)(t.m0 + row) * a.out + col) =
                            *reinterpret_cast<const u32x4q *>(lds.x + buf + row * 128 + ((chunk ^ (row & 7)) << 4));
                }
            } else {
                constexpr uint32_t B = MODE == F32OUT ? 4 : 2;              // bytes of a value
                constexpr int P = MODE == F32OUT ? 1 : 2, C = 4 * B;        // token tiles and chunks of a row in 4 KiB
                if (a.out % (16 / B) || (reinterpret_cast<uintptr_t>(a.y) & 15u)) {  // rows that start unaligned
                    uint32_t to[NS];
#pragma unroll
                    for (int i = 0; i < NS; i++) to[i] = lds.map[s][32 * i + 16 * tg + c];
                    store_rows<MODE, 4, NS>(a, acc, to, ct * 256 + wg * 64 + 16 * q);
                    return;
                }
                uint8_t *const mine = lds.w + 2 * buf + 4096 * wv;  // of this wave alone
#pragma unroll
                for (int h = 0; h < NS; h += P) {
#pragma unroll
                    for (int i = h; i < min(h + P, NS); i++) {
                        uint8_t *const row = mine + (16 * (i - h) + c) * (16 * C);
#pragma unroll
                        for (int k = 0; k < C / 4; k++) {
                            u32x4q v;
                            if constexpr (MODE == F32OUT) {
                                v = __builtin_bit_cast(u32x4q, acc[k][i]);
                            } else {
                                const f32x4q lo = acc[2 * k][i], hi = acc[2 * k + 1][i];
                                v = u32x4q{bf16_pair(lo[0], lo[1]), bf16_pair(lo[2], lo[3]), bf16_pair(hi[0], hi[1]),
                                           bf16_pair(hi[2], hi[3])};
                            }
                            *reinterpret_cast<u32x4q *>(row + (((C / 4 * q + k) ^ (c & (C - 1))) << 4)) = v;
                        }
                    }
                    wave_lds_sync();
#pragma unroll
                    for (int m = 0; m < 16 * P * C / 64; m++) {
                        const uint32_t r = (64 * m + lane) / C, chunk = lane % C;  // row of the staged ones
                        const int i = h + m * (64 / C) / 16;
                        const uint32_t col = ct * 256 + wg * 64 + chunk * (16 / B);
                        if (i >= NS) continue;
                        const u32x4q v = *reinterpret_cast<const u32x4q *>(mine + r * (16 * C) + ((chunk ^ (r & (C - 1))) << 4));
                        const uint32_t to = lds.map[s][32 * i + 16 * tg + r % 16];
                        if (to != 0xffffffffu && col < a.out)
                            *reinterpret_cast<u32x4q *>(static_cast<uint8_t *>(a.y) + ((uint64_t)to * a.out + col) * B) = v;
                    }
                    wave_lds_sync();
                }
            }
        };
        // slot s over the first NS token tiles of each wave
        auto item = [&](auto tiles, uint32_t s) {
            constexpr int NS = decltype(tiles)::value;
            f32x4q acc[4][NS] = {};
            // (the item's first step is in LDS since the last item's last step began)
            Codes wc[4], xc[NS];
            Scales sc;
#pragma unroll
            for (int j = 0; j < 4; j++) wc[j] = weights(cur, j);
#pragma unroll
            for (int i = 0; i < NS; i++) xc[i] = tokens(cur, i);
            scales(sc, slot0);
            uint32_t slot = slot0 + 1;
            // the step's loads go where its own rows were: they are read out
            auto step = [&](bool loads, bool last) {
                begin();
                compute(acc, wc, xc, sc, next, slot, last, [&](int i) {
                    if (loads) load_part(i, cur);
                });
                slot = (slot + 1) % kScaleSlots;
                cur = next;
                next = next == 2 * kStage ? 0 : next + kStage;
            };
            for (uint32_t kb = 0; kb + 1 < nk; kb++) step(true, false);
            // where the last step's loads would go, the outputs are first: they
            // leave through it in whole lines
            const uint32_t spare = cur;
            step(false, true);
            slot0 = (slot0 + (nk + kGroup - 1) / kGroup * kGroup) % kScaleSlots;
            __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));
            landed = true;
            outputs(acc, s, spare);
            barrier();
            ahead(spare);
        };
        for (uint32_t s = 0; s < slots; s++) {
            // (every wave takes the same way: the barriers are inside)
            const uint32_t live = __builtin_amdgcn_readfirstlane(lds.slot[s].end - lds.slot[s].m0);
            if (live > 96) item(std::integral_constant<int, 4>{}, s);
            else if (live > 64) item(std::integral_constant<int, 3>{}, s);
            else if (live > 32) item(std::integral_constant<int, 2>{}, s);
            else item(std::integral_constant<int, 1>{}, s);
        }
        __builtin_amdgcn_s_waitcnt(0);  // the loads past the last item have landed
        if (slots < kSlots) return;
        __syncthreads();
    }
}

// ACT's F32 rows in 8 bits, tile by tile as its launch listed them: a block per tile
// and 128 columns, whose 16 lanes hold eight columns of a row each.
constexpr int kQuantThreads = 256;
__global__ __launch_bounds__(kQuantThreads) void quantize_kernel(Args a) {
    const uint32_t tid = threadIdx.x, ob = gridDim.y, col = 128 * blockIdx.y + 8 * (tid % 16);
    const uint32_t m0 = a.list[2 + 2 * blockIdx.x], end = a.list[3 + 2 * blockIdx.x];
    if (blockIdx.x >= a.list[0]) return;
    const bool cols_in = col < a.out;  // (out is a multiple of 16)
    for (uint32_t p = m0 + tid / 16; p < end; p += kQuantThreads / 16) {
        float v[8] = {};
        if (cols_in) {
            const float *const from = static_cast<const float *>(a.y) + (uint64_t)p * a.out + col;
            const f32x4q lo = *reinterpret_cast<const f32x4q *>(from), hi = *reinterpret_cast<const f32x4q *>(from + 4);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = lo[j], v[4 + j] = hi[j];
        }
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, abs_word(v[j]));
        const uint32_t sb = q8_scale_bits(row16_max(top));
        if (!cols_in || (a.perm ? a.perm[p] : p) / a.kdiv >= a.xrows) continue;
        const float r = q8_inverse(sb);
        *reinterpret_cast<u32x2q *>(a.codes + (uint64_t)p * a.out + col) =
            u32x2q{q8_codes4(v[0], v[1], v[2], v[3], r), q8_codes4(v[4], v[5], v[6], v[7], r)};
        if (tid % 16 == 0) a.scales[(uint64_t)p * ob + blockIdx.y] = (uint16_t)sb;
    }
}

}  // namespace q8

// The stream kernel's forms of one mode: its outputs per block and its kernel.
struct Form {
    uint32_t cols, threads;
    void (*kernel)(q8::Args);
};
// Waves of 16 rows, split along the columns until the launch has 1024 of them
// or each two blocks; 32 rows where there are plenty, or few columns to load ahead
// (16 experts of 768 columns to 2048, 128 rows: 7.8 us, with 16 rows 10.2; 512
// experts of 512, 10 rows: 5.3, 7.7).
template <int MODE, int TT>
static Form stream_form(uint32_t out, uint32_t kb, uint64_t tiles) {
    using namespace q8;
    const uint64_t waves = (uint64_t)((out + 15) / 16) * tiles;
    if constexpr (MODE == SWIGLU) {
        return Form{128, 512, stream_kernel<SWIGLU, 2, 1, 1, 8, 2, 4>};
    } else if constexpr (MODE == ACT) {
        if (waves >= 1024 || kb < 4) return Form{64, 256, stream_kernel<ACT, 2, TT, 1, 4, 4, 2>};
        if (waves >= 512 || kb < 8) return Form{32, 256, stream_kernel<ACT, 2, TT, 2, 4, 4, 2>};
        return Form{16, 256, stream_kernel<ACT, 2, TT, 4, 4, 4, 2>};
    } else {
        if (waves >= 2048 || (TT == 1 && waves >= 1024 && kb < 8))
            return Form{128, 256, stream_kernel<MODE, 2, TT, 1, 4, TT == 1 ? 2 : 3, TT == 1 ? 4 : 2>};
        if (waves >= 1024 || kb < 4) return Form{64, 256, stream_kernel<MODE, 1, TT, 1, 4, TT == 1 && MODE == BF16OUT ? 8 : 4, 2>};
        if (waves >= 512 || kb < 8) return Form{32, 256, stream_kernel<MODE, 1, TT, 2, 4, 4, 2>};
        if (waves >= 256 || kb < 16) return Form{16, 256, stream_kernel<MODE, 1, TT, 4, 4, 4, 2>};
        return Form{16, 512, stream_kernel<MODE, 1, TT, 8, 8, 4, 2>};
    }
}

static hipError_t launch_form(Prof *p, hipStream_t s, const char *name, const Form &f, uint64_t tiles, q8::Args a,
                              uint64_t most_blocks = 0x7ffffff8) {
    a.col_tiles = (a.out + f.cols - 1) / f.cols;
    a.tiles = (uint32_t)tiles;
    uint64_t blocks = (tiles * a.col_tiles + q8::kXcds - 1) / q8::kXcds * q8::kXcds;
    if (blocks > 0x7ffffff8ull) return hipErrorInvalidConfiguration;
    if (blocks > most_blocks) blocks = most_blocks;
    if (blocks * f.threads > 0xffffffffull) return hipErrorInvalidConfiguration;  // (2^34 outputs or more, or tiles of few rows)
    return launch_kernel(p, name, f.kernel, dim3((uint32_t)blocks), dim3(f.threads), 0, s, a);
}

template <int MODE>
static hipError_t launch_q8(Prof *p, hipStream_t s, const char *name, q8::Args a) {
    using namespace q8;
    a.kb = (a.in + 127) / 128;
    const uint32_t experts = a.offsets ? a.experts : 1;
    const uint64_t live = experts < a.P ? experts : a.P, cols = MODE == SWIGLU ? 128 : 256, ct = (a.out + cols - 1) / cols;
    // every non-empty segment may end in a partial tile
    auto max_tiles = [&](uint32_t bm) { return a.P / bm + (a.offsets ? live : (uint64_t)(a.P % bm != 0)); };
    // Tiles of 128 rows need CUs to work on them: enough items, or enough rows
    // (2048 columns, microseconds of tiles against the best stream form):
    //   SwiGLU  512 outputs, 1 expert, 512 rows (16 items): 19.1, 15.4;  4 experts, 1024 rows (32): 19.7, 45.9
    //           768 outputs, 16 experts, 16 rows (96 items): 15.3, 12.5;  128 rows: 15.6, 17.8;  256 rows: 15.7, 28.0
    //           512 outputs, 512 experts, 20 rows (80 items): 15.7, 16.2;  40 rows (160): 19.6, 24.7
    //   bf16    4096 outputs, 128 rows (16 items): 16.0, 13.2;  256 rows (32): 16.4, 19.1
    //           16384 outputs, 32 rows (64 items): 13.7, 13.6;  48 rows: 13.8, 19.4
    //   F32     4096 outputs, 256 rows (32 items): 31.5, 20.3;  512 rows (64): 33.5, 38.3
    // and an expert's rows to be worth its steps (768 columns to 2048, 64 experts):
    //   bf16    512 rows: 21.3, 18.7;  1024: 21.7, 24.9      F32  512 rows: 23.5, 19.6;  1024: 24.1, 26.1
    // SwiGLU's steps are worth it from the first row on (2048 to 512, 64 experts, 64 rows: 20.4, 24.7;
    // 512 experts, 640 rows: 131, 129).
    // DMA offsets and the scales' indexes there are 32-bit.
    constexpr uint64_t kRows = MODE == SWIGLU ? 0 : MODE == F32OUT ? 16 : 12;
    const bool fills = ct * a.P >= (MODE == SWIGLU ? kQ8FewRows : MODE == F32OUT ? 5120 : 2560) || (MODE == BF16OUT && ct * live >= 80) ||
                       (MODE == SWIGLU && ct * (a.P + 32 * live) >= kQ8FewWork);
    const bool tiled = fills && a.P >= kRows * experts && (uint64_t)a.xrows * a.in < 0xffffffffull &&
                       (uint64_t)a.out * a.in < 0xffffffffull &&
                       (uint64_t)experts * ((a.out + 127) / 128) * a.kb < 0xffffffffull;
    // Two token tiles a wave read the weights half as often, where that leaves 256
    // waves (24 rows, 2048 columns to 4096: 5.1 us against 6.2; 4096 to 2048: 7.6 against 6.3)
    const bool two = a.P > 16ull * experts && (uint64_t)((a.out + 15) / 16) * ((a.P + 15) / 16) >= 512;
    if (tiled)
        return launch_form(p, s, name, Form{(uint32_t)cols, 512, a.in % 128 ? tile_kernel<MODE, true> : tile_kernel<MODE, false>},
                           max_tiles(128), a, kCus);
    const uint64_t tiles = max_tiles(two ? 32 : 16);
    if constexpr (MODE == SWIGLU) {
        // A scale needs 128 outputs: blocks that hold them (512 KiB of weights at
        // 2048 columns) are few, so blocks of 16 to 64 write F32 rows and a second
        // launch quantises them (10 rows of 512 experts: 20.2 us, 12.1).  One launch
        // whose last block of each 128 quantises took 11.1 where the rows' order
        // rested on their stores having landed; 14.2 with a release and an acquire
        // around the count, which write back and drop a whole L2.  (What does not
        // fit has 2^32 bytes of rows or weights.)
        if ((uint64_t)a.P * a.out <= kQ8RowsLen && tiles <= kQ8TilesLen) {
            const hipError_t e = launch_form(
                p, s, name, two ? stream_form<ACT, 2>(a.out, a.kb, tiles) : stream_form<ACT, 1>(a.out, a.kb, tiles), tiles, a);
            if (e != hipSuccess) return e;
            return launch_kernel(p, "quantize_q8", quantize_kernel, dim3((uint32_t)tiles, (a.out + 127) / 128),
                                 dim3(kQuantThreads), 0, s, a);
        }
        return launch_form(p, s, name, stream_form<SWIGLU, 1>(a.out, a.kb, max_tiles(16)), max_tiles(16), a);
    } else {
        return launch_form(p, s, name, two ? stream_form<MODE, 2>(a.out, a.kb, tiles) : stream_form<MODE, 1>(a.out, a.kb, tiles),
                           tiles, a);
    }
}

hipError_t launch_q8_rows(Prof *p, hipStream_t s, const char *name, const Q8Weight &w, const Q8Rows &x,
                          const uint32_t *offsets, const uint32_t *perm, void *y, bool bf16) {
    q8::Args a{};
    a.w = w.codes, a.ws = w.scales, a.stype = w.stype, a.in = w.in, a.out = w.out, a.experts = w.experts;
    a.x = x.codes, a.xs = x.scales, a.xrows = x.rows, a.P = x.rows;
    a.offsets = offsets, a.perm = perm, a.y = y, a.kdiv = 1;
    return bf16 ? launch_q8<q8::BF16OUT>(p, s, name, a) : launch_q8<q8::F32OUT>(p, s, name, a);
}

hipError_t launch_q8_swiglu(Prof *p, hipStream_t s, const Q8Weight &gate, const Q8Weight &up, const Q8Rows &x,
                            const uint32_t *offsets, const uint32_t *perm, uint32_t k, const Q8Rows &out,
                            float *rows) {
    q8::Args a{};
    a.w = gate.codes, a.ws = gate.scales, a.w2 = up.codes, a.ws2 = up.scales, a.stype = gate.stype;
    a.in = gate.in, a.out = gate.out, a.experts = gate.experts;
    a.x = x.codes, a.xs = x.scales, a.xrows = x.rows, a.P = out.rows;
    a.offsets = offsets, a.perm = perm, a.kdiv = k;
    a.codes = out.codes, a.scales = out.scales;
    a.y = rows, a.list = reinterpret_cast<uint32_t *>(rows + kQ8RowsLen);
    return launch_q8<q8::SWIGLU>(p, s, "expert_swiglu_q8", a);
}

}  // namespace moehip
