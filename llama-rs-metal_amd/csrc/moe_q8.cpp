// C entries of the 8-bit floating point operators (include/moe_hip.h): checks,
// then one launch each (two for a SwiGLU of few positions).  No counterpart in the reference, whose weights are
// affine, GGML or dense.
#include "abi_common.hpp"

namespace {

uint64_t blocks128(uint64_t n) { return (n + 127) / 128; }
bool aligned(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
bool has(const moe_buffer &b) { return b.ptr != nullptr && b.len != 0; }
// a * b, UINT64_MAX when it overflows
uint64_t mul(uint64_t a, uint64_t b) { return b && a > UINT64_MAX / b ? UINT64_MAX : a * b; }

moe_status check_weight_q8(moe_gpu *g, const moe_weight *w, uint32_t ndims, const char *what) {
    const std::string n = what;
    if (!w) return shape(g, n + ": missing weight");
    if (w->dtype != MOE_E4M3 || w->bits != 0) return shape(g, n + ": the weight is not MOE_E4M3");
    if (w->ndims != ndims) return shape(g, n + ": tensor dimensions");
    const uint64_t in = w->dims[0], out = w->dims[1], e = ndims > 2 ? w->dims[2] : 1;
    if (in == 0 || out == 0 || e == 0) return shape(g, n + ": tensor dimensions");
    if (in % 16) return shape(g, n + ": rows must be a multiple of 16 values");
    if (in > (1u << 24) || out > 0x7fffffffull || e > 16384) return shape(g, n + ": size limit");
    if (w->group_size != 128 || !float_type(w->scale_type))
        return shape(g, n + ": scales per 128 x 128 block in F32, F16 or BF16");
    if (w->data.bytes != mul(mul(in, out), e) ||
        w->scales.bytes != e * blocks128(out) * blocks128(in) * scalar_bytes(w->scale_type))
        return shape(g, n + ": code/scale length");
    if (!aligned(w->data.ptr, 16) || !aligned(w->scales.ptr, scalar_bytes(w->scale_type)))
        return shape(g, n + ": codes must be 16-byte aligned");
    return check_own(g, {rng(w->data), rng(w->scales)});
}

moe_status check_rows8(moe_gpu *g, const moe_rows8 &r, const char *what) {
    const std::string n = what;
    if (r.rows == 0 || r.n == 0 || r.n % 16) return shape(g, n + ": 8-bit rows of a multiple of 16 values");
    if (r.rows > 0x7fffffffull || r.n > (1u << 24)) return shape(g, n + ": size limit");
    if (r.codes.bytes != r.rows * r.n || r.scales.bytes != r.rows * blocks128(r.n) * 2)
        return shape(g, n + ": code/scale length");
    if (!aligned(r.codes.ptr, 16) || !aligned(r.scales.ptr, 2)) return shape(g, n + ": codes must be 16-byte aligned");
    return check_own(g, {rng(r.codes), rng(r.scales)});
}

Q8Weight q8_weight(const moe_weight &w) {
    return Q8Weight{static_cast<const uint8_t *>(w.data.ptr), w.scales.ptr, w.scale_type, (uint32_t)w.dims[0],
                    (uint32_t)w.dims[1], w.ndims > 2 ? (uint32_t)w.dims[2] : 1u};
}
Q8Rows q8_rows(const moe_rows8 &r) {
    return Q8Rows{static_cast<uint8_t *>(const_cast<void *>(r.codes.ptr)),
                  static_cast<uint16_t *>(const_cast<void *>(r.scales.ptr)), (uint32_t)r.rows, (uint32_t)r.n};
}

// y of `values` values of `type` (F32, or BF16 two per element)
moe_status check_values(moe_gpu *g, const moe_buffer &y, uint32_t type, uint64_t values, const char *what) {
    const std::string n = what;
    if (type != MOE_F32 && type != MOE_BF16) return shape(g, n + ": values of F32 or BF16");
    if (type == MOE_BF16 ? values % 2 || y.len != values / 2 : y.len != values) return shape(g, n + ": length");
    if (!aligned(y.ptr, 4)) return shape(g, n + ": alignment");
    return check_own(g, {rng(y)});
}

}  // namespace

extern "C" {

moe_status moe_norm_q8(moe_gpu *g, moe_buffer x, moe_buffer residual, const moe_weight *w, moe_buffer sum,
                       moe_buffer y, moe_rows8 q, float eps) {
    moe_status st = need_batch(g);
    if (st) return st;
    if (!w || w->bits) return shape(g, "RMSNorm weights must be floating point");
    if ((st = check_weight(g, w, "norm"))) return st;
    if ((st = check_rows8(g, q, "norm"))) return st;
    const uint64_t len = q.rows * q.n;
    if (w->ndims != 1 || w->dims[0] != q.n || x.len != len || (has(residual) && residual.len != len) ||
        (has(sum) && sum.len != len) || (has(y) && y.len != len) || !std::isfinite(eps) || eps <= 0.f)
        return shape(g, "norm");
    if (!aligned(x.ptr, 4) || !aligned(residual.ptr, 4) || !aligned(sum.ptr, 4) || !aligned(y.ptr, 4))
        return shape(g, "norm: alignment");
    std::vector<Range> reads{rng(x), rng(w->data)}, writes{rng(q.codes), rng(q.scales)};
    if ((st = check_own(g, {rng(x)}))) return st;
    if (has(residual)) {
        if ((st = check_own(g, {rng(residual)}))) return st;
        reads.push_back(rng(residual));
    }
    if (has(y)) {
        if ((st = check_own(g, {rng(y)}))) return st;
        writes.push_back(rng(y));
    }
    if ((st = check_alias(g, reads, writes, false))) return st;
    if (has(sum)) {
        // the sum may replace x or the residual exactly
        if ((st = check_own(g, {rng(sum)}))) return st;
        for (const Range &o : writes)
            if (overlaps(o, rng(sum))) return shape(g, "overlapping GPU outputs");
        if (overlaps(rng(sum), rng(w->data))) return shape(g, "GPU input/output alias");
        if ((st = check_alias(g, {rng(x)}, {rng(sum)}, true))) return st;
        if (has(residual) && (st = check_alias(g, {rng(residual)}, {rng(sum)}, true))) return st;
    }
    const Q8Rows o = q8_rows(q);
    return launched(g, launch_norm_q8(&g->prof, g->stream, (const float *)x.ptr,
                                      has(residual) ? (const float *)residual.ptr : nullptr, w->data.ptr, w->dtype,
                                      has(sum) ? (float *)sum.ptr : nullptr, has(y) ? (float *)y.ptr : nullptr,
                                      o.codes, o.scales, o.rows, o.n, eps),
                    "norm_q8");
}

moe_status moe_matmul_q8(moe_gpu *g, const moe_weight *w, moe_rows8 x, moe_buffer y, uint32_t y_type) {
    moe_status st = need_batch(g);
    if (st) return st;
    if ((st = check_weight_q8(g, w, 2, "matmul"))) return st;
    if ((st = check_rows8(g, x, "matmul"))) return st;
    if (x.n != w->dims[0]) return shape(g, "matmul shape");
    if ((st = check_values(g, y, y_type, x.rows * w->dims[1], "matmul output"))) return st;
    if ((st = check_alias(g, {rng(w->data), rng(w->scales), rng(x.codes), rng(x.scales)}, {rng(y)}, false)))
        return st;
    return launched(g, launch_q8_rows(&g->prof, g->stream, "matmul_q8", q8_weight(*w), q8_rows(x), nullptr, nullptr,
                                      y.ptr, y_type == MOE_BF16),
                    "matmul_q8");
}

moe_status moe_expert_matmul_q8(moe_gpu *g, const moe_weight *w, moe_rows8 x, moe_buffer offsets, moe_buffer perm,
                                moe_buffer y, uint32_t y_type) {
    moe_status st = need_batch(g);
    if (st) return st;
    if ((st = check_weight_q8(g, w, 3, "expert matmul"))) return st;
    if ((st = check_rows8(g, x, "expert matmul"))) return st;
    if (x.n != w->dims[0] || offsets.len != w->dims[2] + 1 || (has(perm) && perm.len != x.rows))
        return shape(g, "expert matmul");
    if (!aligned(offsets.ptr, 4) || !aligned(perm.ptr, 4)) return shape(g, "expert matmul: alignment");
    if ((st = check_values(g, y, y_type, x.rows * w->dims[1], "expert matmul output"))) return st;
    std::vector<Range> reads{rng(w->data), rng(w->scales), rng(x.codes), rng(x.scales), rng(offsets)};
    if ((st = check_own(g, {rng(offsets)}))) return st;
    if (has(perm)) {
        if ((st = check_own(g, {rng(perm)}))) return st;
        reads.push_back(rng(perm));
    }
    if ((st = check_alias(g, reads, {rng(y)}, false))) return st;
    return launched(g, launch_q8_rows(&g->prof, g->stream, "expert_matmul_q8", q8_weight(*w), q8_rows(x),
                                      (const uint32_t *)offsets.ptr, has(perm) ? (const uint32_t *)perm.ptr : nullptr,
                                      y.ptr, y_type == MOE_BF16),
                    "expert_matmul_q8");
}

moe_status moe_expert_swiglu_q8(moe_gpu *g, const moe_weight *gate, const moe_weight *up, moe_rows8 x,
                                moe_buffer offsets, moe_buffer perm, uint64_t k, moe_rows8 q) {
    moe_status st = need_batch(g);
    if (st) return st;
    if ((st = check_weight_q8(g, gate, 3, "expert gates")) || (st = check_weight_q8(g, up, 3, "expert ups")))
        return st;
    if ((st = check_rows8(g, x, "expert input")) || (st = check_rows8(g, q, "expert output"))) return st;
    for (int i = 0; i < 3; i++)
        if (gate->dims[i] != up->dims[i]) return shape(g, "expert ups dimensions");
    if (gate->scale_type != up->scale_type) return shape(g, "expert gates and ups: scales of one type");
    if (k == 0 || !fits_u32(k) || x.n != gate->dims[0] || q.n != gate->dims[1] || offsets.len != gate->dims[2] + 1 ||
        (has(perm) ? perm.len != q.rows || mul(x.rows, k) != q.rows : k != 1 || q.rows != x.rows))
        return shape(g, "expert swiglu");
    if (!aligned(offsets.ptr, 4) || !aligned(perm.ptr, 4)) return shape(g, "expert swiglu: alignment");
    std::vector<Range> reads{rng(gate->data), rng(gate->scales), rng(up->data), rng(up->scales),
                             rng(x.codes),    rng(x.scales),     rng(offsets)};
    if ((st = check_own(g, {rng(offsets)}))) return st;
    if (has(perm)) {
        if ((st = check_own(g, {rng(perm)}))) return st;
        reads.push_back(rng(perm));
    }
    if ((st = check_alias(g, reads, {rng(q.codes), rng(q.scales)}, false))) return st;
    return launched(g, launch_q8_swiglu(&g->prof, g->stream, q8_weight(*gate), q8_weight(*up), q8_rows(x),
                                        (const uint32_t *)offsets.ptr,
                                        has(perm) ? (const uint32_t *)perm.ptr : nullptr, (uint32_t)k, q8_rows(q),
                                        g->q8_rows),
                    "expert_swiglu_q8");
}

moe_status moe_mix_tokens(moe_gpu *g, moe_buffer x, uint32_t x_type, moe_buffer w, moe_buffer residual, moe_buffer y,
                          uint64_t tokens) {
    moe_status st = need_batch(g);
    if (st) return st;
    if (tokens == 0 || w.len == 0 || y.len == 0 || w.len % tokens || y.len % tokens) return shape(g, "mix");
    const uint64_t k = w.len / tokens, h = y.len / tokens;
    if (!fits_u32(tokens) || !fits_u32(k) || !fits_u32(h)) return shape(g, "dimension exceeds u32");
    if (has(residual) && residual.len != y.len) return shape(g, "mix");
    if ((st = check_values(g, x, x_type, mul(mul(tokens, k), h), "mix input"))) return st;
    if (!aligned(w.ptr, 4) || !aligned(residual.ptr, 4) || !aligned(y.ptr, 4)) return shape(g, "mix: alignment");
    if ((st = check_own(g, {rng(w), rng(y)}))) return st;
    if ((st = check_alias(g, {rng(x), rng(w)}, {rng(y)}, false))) return st;
    if (has(residual)) {
        if ((st = check_own(g, {rng(residual)}))) return st;
        if ((st = check_alias(g, {rng(residual)}, {rng(y)}, true))) return st;  // y may be the residual itself
    }
    return launched(g, launch_mix_tokens(&g->prof, g->stream, x.ptr, x_type == MOE_BF16, (const float *)w.ptr,
                                         has(residual) ? (const float *)residual.ptr : nullptr, (float *)y.ptr,
                                         (uint32_t)tokens, (uint32_t)k, (uint32_t)h),
                    "mix_tokens");
}

}  // extern "C"
