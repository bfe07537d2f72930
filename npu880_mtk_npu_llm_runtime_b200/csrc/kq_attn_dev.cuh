// kq_attn_dev.cuh -- device code shared by the attention kernels.
#pragma once

#include "kq_common.cuh"
#include "kq_attn.h"

namespace kq {

__device__ __forceinline__ float2 h2_to_f2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
__device__ __forceinline__ uint32_t f2_to_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Two weighted means as fp16.  The weights of the sum of values were rounded to fp16 and those of the sum of weights
// were not, so a mean of values near fp16's largest may lie up to 2^-11 beyond it: it stands for the largest, as no
// mean is larger than its values.  (This form takes an infinity for the largest too; mean_to_h2 keeps it.)
__device__ __forceinline__ uint32_t finite_mean_to_h2(float a, float b) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t mean_to_h2(float a, float b) {
    auto held = [](float x) { return fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x; };
    return f2_to_h2(held(a), held(b));
}

// No weight, and no factor of what was summed before, is less than this: a value that is infinite stays so under
// a weight that would vanish (0 times it is NaN), and to finite ones it adds nothing that fp32 holds.  (A score
// of -inf has the weight 0; NaN stays.)
constexpr float kLeast = 1.17549435e-38f;  // fp32's smallest normal number
__device__ __forceinline__ float at_least(float w, float least) { return w < least ? least : w; }

// One more arrival at a counter other CTAs count on too: releases this thread's (and, after a barrier,
// its CTA's) writes, acquires those of the arrivals before it, whose number it returns.
__device__ __forceinline__ unsigned count_arrival(unsigned *count) {
    unsigned n;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(n) : "l"(count) : "memory");
    return n;
}

// The page that holds position j of sequence seq, or -1 (and an error) where the table names none.
__device__ __forceinline__ int kv_page(const KvView &c, int seq, int j, int *status) {
    const int page = c.table[(long long)seq * c.table_stride + (j >> c.page_shift)];
    if (kv_page_ok(c, page)) return page;
    report_error(status, DEV_ERR_CACHE);
    return -1;
}

// One row of one head by a warp: out = sum_j softmax_j(scale q.k_j) v_j over exactly the keys of
// `span`, everything in fp32, 32 keys at a time: a lane takes a key for the scores, and values
// [lane D/32, (lane + 1) D/32) of the row for the sum.  No key outside the span is read.
template <int D>
__device__ __noinline__ void attn_row(const KvView &c, int seq, int kv_head, KvSpan span, const uint16_t *q,
                                      uint16_t *out, float scale, int lane, int *status) {
    constexpr int W = D / 64;  // 32-bit words of a row per lane
    constexpr int U = 8;       // rows of V on their way at once
    float2 acc[W];
    const int mask = (1 << c.page_shift) - 1;
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = make_float2(0.0f, 0.0f);
    float m = -INFINITY, sum = 0.0f;  // sum: this lane's keys
    const int n = kv_count(span);
    bool seen = false;
    for (int e0 = 0; e0 < n; e0 += 32) {
        long long at = -1;
        float s = 0.0f;
        if (e0 + lane < n) {
            const int j = kv_nth(span, e0 + lane), page = kv_page(c, seq, j, status);
            if (page >= 0) at = kv_row(c, page, kv_head, j & mask);
        }
        if (at >= 0) {
#pragma unroll 4
            for (int i = 0; i < D / 8; ++i) {
                const uint4 k = *reinterpret_cast<const uint4 *>(c.k + at + 8 * i);
                const uint4 x = *reinterpret_cast<const uint4 *>(q + 8 * i);
                const uint32_t kw[4] = {k.x, k.y, k.z, k.w}, xw[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float2 a = h2_to_f2(kw[u]), b = h2_to_f2(xw[u]);
                    s = fmaf(a.x, b.x, fmaf(a.y, b.y, s));
                }
            }
            s = __fmul_rn(s, scale);  // (one value: contracted into s - top below, large scores would not cancel)
        }
        const uint32_t there = __ballot_sync(0xffffffffu, at >= 0);
        seen |= there != 0;
        float top = at >= 0 ? s : -INFINITY;
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        top = fmaxf(m, top);
        // before the first score above -inf there is nothing to rescale; a NaN score stays NaN
        const float old = (m == -INFINITY) ? 1.0f : at_least(__expf(m - top), kLeast);
        const float w = (at < 0 || s == -INFINITY) ? 0.0f : at_least(__expf(s - top), kLeast);
        m = top;
        sum = sum * old + w;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            acc[i].x *= old;
            acc[i].y *= old;
        }
        for (int i0 = 0; i0 < 32 && (there >> i0); i0 += U) {
            uint32_t v[U][W];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long row = __shfl_sync(0xffffffffu, at, i0 + u);
#pragma unroll
                for (int i = 0; i < W; ++i)
                    v[u][i] = row >= 0 ? reinterpret_cast<const uint32_t *>(c.v + row)[lane * W + i] : 0u;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float wu = __shfl_sync(0xffffffffu, w, i0 + u);
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const float2 x = h2_to_f2(v[u][i]);
                    acc[i].x = fmaf(wu, x.x, acc[i].x);
                    acc[i].y = fmaf(wu, x.y, acc[i].y);
                }
            }
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const float inv = seen ? 1.0f / sum : 0.0f;  // scores all -inf: 0 / 0, NaN as in the formula
#pragma unroll
    for (int i = 0; i < W; ++i)
        reinterpret_cast<uint32_t *>(out)[lane * W + i] = seen ? mean_to_h2(acc[i].x * inv, acc[i].y * inv) : 0u;
}

}  // namespace kq
