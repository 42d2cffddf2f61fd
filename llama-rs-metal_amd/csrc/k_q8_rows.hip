// Row operators around the 8-bit products: the RMSNorm that takes the residual
// in and writes 8-bit rows, and the weighted sum of each token's expert rows.
#include "q8.hpp"

namespace moehip {

// s = x + residual; y = s / sqrt(mean(s^2) + eps) * w; per 128 columns
// scale = bf16(max|y| / 448), code = e4m3(y / scale).
//
// One block per row; a thread holds groups of eight columns, so 16 lanes (one
// DPP row) hold the 128 columns that share a scale.  Rows of up to
// kQ8NormHold * 2048 columns are read once and stay in registers between the sum
// of squares and the output; longer ones are read again (as s, from `sum`
// where that is written: it may be x or the residual itself).
//
// Bound by its bytes: 4096 rows of 2048 with residual, sum and F32 rows, 143 MB in
// 33.9 us or 4.2 TB/s, where a copy reaches 4.65; one row takes an empty launch's 4 us.
// (`y` shows v, so its codes are those of the true F32 quotient: divisions, 33.9 us,
// where products with a reciprocal took 33.8 and missed quotients between two codes.)
constexpr uint32_t kQ8NormThreads = 256, kQ8NormHold = 2;

template <int T, bool VEC>
__global__ __launch_bounds__(kQ8NormThreads) void norm_q8_kernel(const float *x, const float *resid, const void *w,
                                                                 float *sum, float *y, uint8_t *codes,
                                                                 uint16_t *scales, uint32_t rows, uint32_t n, float eps) {
    __shared__ float part[kQ8NormThreads / 64];
    const uint32_t row = blockIdx.y * gridDim.x + blockIdx.x, tid = threadIdx.x, step = 8 * kQ8NormThreads;
    if (row >= rows) return;
    const uint64_t base = (uint64_t)row * n;
    auto load = [&](const float *p, uint32_t i, float *v) {
        if constexpr (VEC) {
            const f32x4q a = *reinterpret_cast<const f32x4q *>(p + base + i);
            const f32x4q b = *reinterpret_cast<const f32x4q *>(p + base + i + 4);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = a[j], v[4 + j] = b[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = p[base + i + j];
        }
    };
    auto store = [&](float *p, uint32_t i, const float *v) {
        if constexpr (VEC) {
            *reinterpret_cast<f32x4q *>(p + base + i) = f32x4q{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4q *>(p + base + i + 4) = f32x4q{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) p[base + i + j] = v[j];
        }
    };
    // s of eight columns, stored where asked; its squares added to `acc`
    auto first = [&](uint32_t i, float *v, float &acc) {
        load(x, i, v);
        if (resid) {
            float r[8];
            load(resid, i, r);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] += r[j];
        }
        if (sum) store(sum, i, v);
#pragma unroll
        for (int j = 0; j < 8; j++) acc += v[j] * v[j];
    };
    float hold[kQ8NormHold][8] = {};
    float acc = 0.f;
#pragma unroll
    for (uint32_t q = 0; q < kQ8NormHold; q++)
        if (8 * tid + q * step < n) first(8 * tid + q * step, hold[q], acc);
    for (uint64_t i = 8 * tid + kQ8NormHold * step; i < n; i += step) {
        float v[8];
        first((uint32_t)i, v, acc);
    }
    acc = wave_sum(acc);
    if ((tid & 63) == 0) part[tid >> 6] = acc;
    __syncthreads();
    acc = (part[0] + part[1]) + (part[2] + part[3]);
    const float inv = 1.0f / sqrtf(acc / (float)n + eps);
    const uint32_t nb = (n + 127) / 128;
    // all 16 lanes of a group come here together (columns past n hold zeros)
    auto finish = [&](uint32_t i, const float *v, bool live) {
        float o[8];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            o[j] = live ? v[j] * inv * load_scalar<T>(w, i + j) : 0.f;
            top = max(top, abs_word(o[j]));
        }
        top = row16_max(top);
        const uint32_t sb = q8_scale_bits(top);
        const float scale = bf16_to_f32(sb);
        if (!live) return;
        if (y) store(y, i, o);
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] /= scale;
        *reinterpret_cast<u32x2q *>(codes + base + i) =
            u32x2q{q8_codes4(o[0], o[1], o[2], o[3]), q8_codes4(o[4], o[5], o[6], o[7])};
        if ((tid & 15) == 0) scales[(uint64_t)row * nb + i / 128] = (uint16_t)sb;
    };
#pragma unroll
    for (uint32_t q = 0; q < kQ8NormHold; q++) {
        const uint32_t i = 8 * tid + q * step;
        if ((i & ~127u) < n) finish(i, hold[q], i < n);
    }
    for (uint64_t i = 8 * tid + kQ8NormHold * step; (i & ~127ull) < n; i += step) {
        float v[8] = {};
        const bool live = i < n;
        if (live) {
            load(sum ? sum : x, (uint32_t)i, v);
            if (resid && !sum) {
                float r[8];
                load(resid, (uint32_t)i, r);
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] += r[j];
            }
        }
        finish((uint32_t)i, v, live);
    }
}

hipError_t launch_norm_q8(Prof *p, hipStream_t s, const float *x, const float *resid, const void *w, uint32_t wtype,
                          float *sum, float *y, uint8_t *codes, uint16_t *scales, uint32_t rows, uint32_t n,
                          float eps) {
    // 16-byte accesses where the F32 arrays start 16-byte aligned (n is a multiple of 16)
    const uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(resid) |
                          reinterpret_cast<uintptr_t>(sum) | reinterpret_cast<uintptr_t>(y);
    const bool vec = (all & 15u) == 0;
    auto kern = vec ? (wtype == 0   ? norm_q8_kernel<0, true>
                       : wtype == 1 ? norm_q8_kernel<1, true>
                                    : norm_q8_kernel<30, true>)
                    : (wtype == 0   ? norm_q8_kernel<0, false>
                       : wtype == 1 ? norm_q8_kernel<1, false>
                                    : norm_q8_kernel<30, false>);
    // a launch has fewer than 2^32 threads along x
    const uint32_t wide = rows < (1u << 22) ? rows : 1u << 22;
    return launch_kernel(p, "norm_q8", kern, dim3(wide, (rows + wide - 1) / wide), dim3(kQ8NormThreads), 0, s, x, resid,
                         w, sum, y, codes, scales, rows, n, eps);
}

// y[t, i] = sum_k w[t, k] * x[t K + k, i] (k ascending) (+ resid[t, i])
//
// Bound by its bytes: 4096 tokens of 10 bf16 rows of 2048 and a residual, 235 MB in
// 44.5 us or 5.3 TB/s.  A thread holds four columns and walks the K rows, so that
// neighbouring lanes read neighbouring bytes of one row and no sum is shared.
constexpr uint32_t kMixThreads = 256;

template <bool BF16, bool VEC>
__global__ __launch_bounds__(kMixThreads) void mix_tokens_kernel(const void *__restrict__ x,
                                                                 const float *__restrict__ w, const float *resid,
                                                                 float *y, uint32_t K, uint32_t h, uint64_t n) {
    constexpr uint32_t V = VEC ? 4 : 1;
    for (uint64_t g = (uint64_t)blockIdx.x * kMixThreads + threadIdx.x; g * V < n;
         g += (uint64_t)gridDim.x * kMixThreads) {
        const uint64_t t = g * V / h;
        const uint32_t i = (uint32_t)(g * V - t * h);
        float acc[V] = {};
        for (uint32_t k = 0; k < K; k++) {
            const float wk = w[t * K + k];
            const uint64_t at = (t * K + k) * h + i;
            if constexpr (VEC && BF16) {
                const u32x2q v = *reinterpret_cast<const u32x2q *>(static_cast<const uint16_t *>(x) + at);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    acc[j] = fmaf(bf16_to_f32((v[j / 2] >> (16 * (j % 2))) & 0xffffu), wk, acc[j]);
            } else if constexpr (VEC) {
                const f32x4q v = *reinterpret_cast<const f32x4q *>(static_cast<const float *>(x) + at);
#pragma unroll
                for (int j = 0; j < 4; j++) acc[j] = fmaf(v[j], wk, acc[j]);
            } else {
                acc[0] = fmaf(load_scalar<BF16 ? 30 : 0>(x, at), wk, acc[0]);
            }
        }
        const uint64_t o = t * h + i;
        if constexpr (VEC) {
            f32x4q r = {0.f, 0.f, 0.f, 0.f};
            if (resid) r = *reinterpret_cast<const f32x4q *>(resid + o);
            *reinterpret_cast<f32x4q *>(y + o) = f32x4q{acc[0] + r[0], acc[1] + r[1], acc[2] + r[2], acc[3] + r[3]};
        } else {
            y[o] = resid ? acc[0] + resid[o] : acc[0];
        }
    }
}

hipError_t launch_mix_tokens(Prof *p, hipStream_t s, const void *x, bool bf16, const float *w, const float *resid,
                             float *y, uint32_t tokens, uint32_t k, uint32_t h) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(resid) |
                          reinterpret_cast<uintptr_t>(y);
    const bool vec = h % 4 == 0 && (all & 15u) == 0;
    const uint64_t n = (uint64_t)tokens * h, groups = vec ? n / 4 : n;
    const uint64_t want = (groups + kMixThreads - 1) / kMixThreads;
    const dim3 grid((uint32_t)(want < (1u << 20) ? want : (1u << 20)));
    auto kern = bf16 ? (vec ? mix_tokens_kernel<true, true> : mix_tokens_kernel<true, false>)
                     : (vec ? mix_tokens_kernel<false, true> : mix_tokens_kernel<false, false>);
    return launch_kernel(p, "mix_tokens", kern, grid, dim3(kMixThreads), 0, s, x, w, resid, y, k, h, n);
}

}  // namespace moehip
