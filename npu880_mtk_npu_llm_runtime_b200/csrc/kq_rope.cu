// kq_rope.cu -- per-head norms, the position rotation and the append to the paged cache.
//
// One kernel for both calls (kq_qk_norm_rope_async, kq_kv_append_async): a head x of D values
// becomes  y = x * gamma / sqrt(mean(x^2) + eps)  and pair (a, b) of y at position p turns by
// t = p * f:  (a cos t - b sin t, a sin t + b cos t).  Values are copied.
#include "kq_common.cuh"
#include "kq_attn.h"

namespace kq {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPasses = 4;  // heads of a row that one CTA takes: up to this many per thread group

struct RowSet {
    const __half *in;
    long long in_stride;
    __half *out;  // nullptr: to the cache
    long long out_stride;
    const __half *gamma;
    int heads;
};

struct RopeParams {
    RowSet q, k, v;  // heads in this order; heads = 0: none
    KvView cache;    // table == nullptr: no append
    const int32_t *seq, *pos;
    int *status;
    float eps;
    int rot, adjacent, passes;
    double turns[KQ_MAX_HEAD_DIM / 2];  // full turns per position: inv_freq / (2 pi)
};

__device__ __forceinline__ float2 h2f(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
__device__ __forceinline__ uint32_t f2h(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Grid: (rows, chunks of heads).  LPH lanes hold a head, 8 values (16 bytes) each, so a warp takes
// 32 / LPH heads and all its loads and stores are whole 16-byte vectors.  cos and sin of a
// position are the same for every head of the row: computed once per CTA into shared memory.
// The angle is p * f / (2 pi) turns in fp64 less its nearest integer (positions of a million keep
// 1e-10 of a turn; fp32 would be off by whole radians), then sin / cos of the fraction in fp32.
template <int D>
__global__ __launch_bounds__(kThreads) void kq_norm_rope(const __grid_constant__ RopeParams p) {
    constexpr int LPH = D / 8;
    constexpr int HPP = kThreads / LPH;  // heads per pass
    __shared__ __align__(16) float s_cos[D / 2], s_sin[D / 2];
    const int tid = threadIdx.x, lane = tid & 31, l = tid % LPH;
    const int row = blockIdx.x;
    pdl_launch_dependents();
    pdl_wait();

    int seq = 0, pos = 0, page = 0;
    if (p.pos) pos = p.pos[row];
    if (p.cache.table) {
        seq = p.seq[row];
        if (seq < 0) return;  // padding (uniform over the CTA)
        bool ok = seq < p.cache.n_seqs && pos >= 0 && pos < kv_reach(p.cache);
        if (ok) {
            page = p.cache.table[(long long)seq * p.cache.table_stride + (pos >> p.cache.page_shift)];
            ok = kv_page_ok(p.cache, page);
        }
        if (!ok) {
            if (tid == 0) report_error(p.status, DEV_ERR_CACHE);
            return;
        }
    }
    const int total = p.q.heads + p.k.heads + p.v.heads;
    const int h0 = blockIdx.y * p.passes * HPP + tid / LPH;

    uint4 x[kMaxPasses];
#pragma unroll
    for (int i = 0; i < kMaxPasses; ++i) {
        const int h = h0 + i * HPP;
        if (i < p.passes && h < total) {
            const RowSet &s = h < p.q.heads ? p.q : h < p.q.heads + p.k.heads ? p.k : p.v;
            const int hh = h < p.q.heads ? h : h < p.q.heads + p.k.heads ? h - p.q.heads : h - p.q.heads - p.k.heads;
            x[i] = *reinterpret_cast<const uint4 *>(s.in + (long long)row * s.in_stride + hh * D + 8 * l);
        } else {
            x[i] = make_uint4(0, 0, 0, 0);
        }
    }
    if (p.rot > 0) {
        if (tid < p.rot / 2) {
            const double u = (double)pos * p.turns[tid];
            float sn, cs;
            sincospif(2.0f * (float)(u - rint(u)), &sn, &cs);
            s_cos[tid] = cs;
            s_sin[tid] = sn;
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kMaxPasses; ++i) {
        if (i >= p.passes) break;
        const int h = h0 + i * HPP;
        const bool have = h < total;
        const bool is_q = h < p.q.heads, is_k = !is_q && h < p.q.heads + p.k.heads;
        const RowSet &s = is_q ? p.q : is_k ? p.k : p.v;
        const int hh = is_q ? h : is_k ? h - p.q.heads : h - p.q.heads - p.k.heads;
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint32_t o[4] = {w[0], w[1], w[2], w[3]};
        // every lane of the warp takes part in the shuffles; a head without work holds zeros
        float ss = 0.0f;
        float2 y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            y[j] = h2f(w[j]);
            ss += y[j].x * y[j].x + y[j].y * y[j].y;
        }
#pragma unroll
        for (int d = 1; d < LPH; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        const int half = p.rot / 2, hc = half / 8;
        int src = l;  // the lane that holds the other values of this lane's pairs
        if (!p.adjacent && 8 * l < p.rot) src = (8 * l < half) ? l + hc : l - hc;
        float2 z[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) z[j] = h2f(__shfl_sync(0xffffffffu, w[j], (lane & ~(LPH - 1)) + src));
        if (!have) continue;
        if (is_q || is_k) {
            if (s.gamma) {
                const float inv = rsqrtf(ss * (1.0f / D) + p.eps);
                const uint4 g = __ldg(reinterpret_cast<const uint4 *>(s.gamma + 8 * l));
                const uint4 gz = __ldg(reinterpret_cast<const uint4 *>(s.gamma + 8 * src));
                const uint32_t gw[4] = {g.x, g.y, g.z, g.w}, gzw[4] = {gz.x, gz.y, gz.z, gz.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 a = h2f(gw[j]), b = h2f(gzw[j]);
                    y[j].x *= inv * a.x;
                    y[j].y *= inv * a.y;
                    z[j].x *= inv * b.x;
                    z[j].y *= inv * b.y;
                }
            }
            if (8 * l < p.rot) {
                if (p.adjacent) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float c = s_cos[4 * l + j], sn = s_sin[4 * l + j];
                        const float2 a = y[j];
                        y[j].x = a.x * c - a.y * sn;
                        y[j].y = a.x * sn + a.y * c;
                    }
                } else {
                    const bool first = 8 * l < half;
                    const int at = first ? 8 * l : 8 * l - half;
                    const float sg = first ? -1.0f : 1.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 c = *reinterpret_cast<const float2 *>(s_cos + at + 2 * j);
                        const float2 sn = *reinterpret_cast<const float2 *>(s_sin + at + 2 * j);
                        y[j].x = y[j].x * c.x + sg * z[j].x * sn.x;
                        y[j].y = y[j].y * c.y + sg * z[j].y * sn.y;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = f2h(y[j].x, y[j].y);
        }
        uint16_t *to;
        if (p.cache.table && !is_q)
            to = (is_k ? p.cache.k : p.cache.v) +
                 kv_row(p.cache, page, hh, pos & ((1 << p.cache.page_shift) - 1)) + 8 * l;
        else
            to = reinterpret_cast<uint16_t *>(s.out) + (long long)row * s.out_stride + hh * D + 8 * l;
        *reinterpret_cast<uint4 *>(to) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

RowSet row_set(const kq_heads *h) {
    RowSet s{};
    if (!h) return s;
    s.in = reinterpret_cast<const __half *>(h->in);
    s.in_stride = (long long)h->in_stride;
    s.out = reinterpret_cast<__half *>(h->out);
    s.out_stride = (long long)h->out_stride;
    s.gamma = reinterpret_cast<const __half *>(h->gamma);
    s.heads = h->heads;
    return s;
}

template <int D>
cudaError_t launch(RopeParams &p, int M, int num_sms, cudaStream_t stream, bool pdl) {
    constexpr int HPP = kThreads / (D / 8);
    const int total = p.q.heads + p.k.heads + p.v.heads;
    const int need = (total + HPP - 1) / HPP;
    p.passes = 1;
    while (p.passes < kMaxPasses && p.passes < need && (long long)M * ((need + p.passes - 1) / p.passes) > 4ll * num_sms)
        ++p.passes;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(M, (need + p.passes - 1) / p.passes);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kq_norm_rope<D>, p);
}

}  // namespace

cudaError_t launch_norm_rope(const RopeLaunch &L, cudaStream_t stream) {
    RopeParams p{};
    p.q = row_set(L.q);
    p.k = row_set(L.k);
    p.v = row_set(L.v);
    if (L.cache) p.cache = *L.cache;
    p.seq = L.seq;
    p.pos = L.pos;
    p.status = L.status;
    p.eps = L.eps;
    if (L.rope && L.rope->rot_dim > 0) {
        p.rot = L.rope->rot_dim;
        p.adjacent = L.rope->style == KQ_ROPE_ADJACENT;
        for (int j = 0; j < p.rot / 2; ++j) p.turns[j] = L.rope->inv_freq[j] * 0.15915494309189533577;  // 1 / (2 pi)
    }
    switch (L.head_dim) {
        case 64: return launch<64>(p, L.M, L.num_sms, stream, L.pdl);
        case 128: return launch<128>(p, L.M, L.num_sms, stream, L.pdl);
        case 256: return launch<256>(p, L.M, L.num_sms, stream, L.pdl);
    }
    return cudaErrorInvalidValue;
}

}  // namespace kq
