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

// One more arrival at a counter other CTAs count on too: releases this thread's (and, after a barrier,
// its CTA's) writes, acquires those of the arrivals before it, whose number it returns.
__device__ __forceinline__ unsigned count_arrival(unsigned *count) {
    unsigned n;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(n) : "l"(count) : "memory");
    return n;
}

// The page that holds position j of sequence seq, or -1 (and an error) where the table names none.
__device__ __forceinline__ int kv_page(const KvView &c, int seq, int j, int *status) {
    const int page = __ldg(c.table + (long long)seq * c.table_stride + (j >> c.page_shift));
    if (kv_page_ok(c, page)) return page;
    report_error(status, DEV_ERR_CACHE);
    return -1;
}

// One row of one head by a warp: out = sum_j softmax_j(scale q.k_j) v_j over exactly the keys of
// `span`, everything in fp32, four keys at a time (lane i holds values [i D/32, (i+1) D/32) of the
// head).  No key outside the span is read.
template <int D>
__device__ __noinline__ void attn_row(const KvView &c, int seq, int kv_head, KvSpan span, const uint16_t *q,
                                      uint16_t *out, float scale, int lane, int *status) {
    constexpr int W = D / 64;  // 32-bit words per lane
    constexpr int U = 4;
    float2 qv[W], acc[W];
    const int mask = (1 << c.page_shift) - 1;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        qv[i] = h2_to_f2(reinterpret_cast<const uint32_t *>(q)[lane * W + i]);
        qv[i].x *= scale;
        qv[i].y *= scale;
        acc[i] = make_float2(0.0f, 0.0f);
    }
    float m = -INFINITY, sum = 0.0f;
    const int n = kv_count(span);
    int seen = 0;  // keys that were there
    for (int e0 = 0; e0 < n; e0 += U) {
        float s[U];
        long long at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            at[u] = -1;
            s[u] = 0.0f;
            if (e0 + u < n) {
                const int j = kv_nth(span, e0 + u);
                const int page = kv_page(c, seq, j, status);
                if (page >= 0) at[u] = kv_row(c, page, kv_head, j & mask) / 2 + lane * W;
            }
            if (at[u] >= 0) {
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const float2 k = h2_to_f2(reinterpret_cast<const uint32_t *>(c.k)[at[u] + i]);
                    s[u] += qv[i].x * k.x + qv[i].y * k.y;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], d);
            if (at[u] < 0) continue;  // uniform over the warp
            ++seen;
            const float mn = fmaxf(m, s[u]);
            // before the first score above -inf there is nothing to rescale; a NaN score stays NaN
            const float old = (m == -INFINITY) ? 0.0f : __expf(m - mn);
            const float w = (s[u] == -INFINITY) ? 0.0f : __expf(s[u] - mn);
            sum = sum * old + w;
            m = mn;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float2 v = h2_to_f2(reinterpret_cast<const uint32_t *>(c.v)[at[u] + i]);
                acc[i].x = acc[i].x * old + w * v.x;
                acc[i].y = acc[i].y * old + w * v.y;
            }
        }
    }
    const float inv = seen ? 1.0f / sum : 0.0f;  // scores all -inf: 0 / 0, NaN as in the formula
#pragma unroll
    for (int i = 0; i < W; ++i)
        reinterpret_cast<uint32_t *>(out)[lane * W + i] = seen ? f2_to_h2(acc[i].x * inv, acc[i].y * inv) : 0u;
}

}  // namespace kq
