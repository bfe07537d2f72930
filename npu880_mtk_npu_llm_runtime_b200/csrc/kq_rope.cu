// kq_rope.cu -- per-head norms, the position rotation and the append to the paged cache.
//
// One kernel for both calls (kq_qk_norm_rope_async, kq_kv_append_async): a head x of D values
// becomes  y = x * gamma / sqrt(mean(x^2) + eps)  and pair (a, b) of y at position p turns by
// t = p * f:  (a cos t - b sin t, a sin t + b cos t).  Values are copied.
#include "kq_attn_dev.cuh"

namespace kq {

namespace {

constexpr int kThreads = 128;
constexpr int kCtasPerSm = 7;  // all rows of a call (4,096 at most) resident at once, one warp each: no second wave
constexpr int kInFlight = 4;  // passes whose loads a lane issues at once, one batch ahead of the arithmetic

struct RowSet {
    const __half *in;
    long long in_stride;
    __half *out;  // nullptr: to the cache
    long long out_stride;
    const __half *gamma;
    int heads;
};

struct RopeParams {
    RowSet q, k, v;  // heads = 0: none
    KvView cache;    // table == nullptr: no append
    const int32_t *seq, *pos;
    int *status;
    float eps;
    int M, rot, adjacent, chunks;
    double turns[KQ_MAX_HEAD_DIM / 2];  // full turns per position: inv_freq / (2 pi)
};

__device__ __forceinline__ uint4 load_row(const __half *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

// A warp takes one row, or (few rows) a chunk of one row's heads; LPH lanes hold a head, 8 values
// (16 bytes) each, so every access is a whole vector and a warp has 32 / LPH heads per pass.
//
// cos and sin of the row's position are the same for all heads: the warp's lanes compute them once
// (the angle is p * f / (2 pi) turns in fp64 less its nearest integer -- positions of a million
// keep 1e-10 of a turn, where fp32 would be off by whole radians -- then the fraction's sine and
// cosine in fp32).  With gamma they make two factors for each of a lane's values x and the other
// value z of its pair: y = (x A + z B) / sqrt(mean(x^2) + eps), so a head costs little more than
// its loads, conversions and the sum of squares.
//
// Bound by the bytes, 2 in and 2 out per value.  4,096 rows of 40 heads of 128 (84 MB): 19 us, 4.4 TB/s; a CTA per row that
// applied gamma, cos and sin to every head took 29; 6 CTAs an SM (more registers, but a second wave of 0.15) 24; batches
// of 2 passes 20.  7 CTAs an SM leave 72 registers a thread, 5 or 6 fewer than the batch ahead wants (20-24 bytes spilled,
// 68-72 loaded again a thread): less than the second wave costs.
template <int D>
__global__ __launch_bounds__(kThreads, kCtasPerSm) void kq_norm_rope(const __grid_constant__ RopeParams p) {
    constexpr int LPH = D / 8, HPP = 32 / LPH;
    __shared__ __align__(16) float s_cos[kThreads / 32][D / 2], s_sin[kThreads / 32][D / 2];
    __shared__ double s_turns[D / 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % LPH, sub = lane / LPH;
    const int task = blockIdx.x * (kThreads / 32) + warp, row = task / p.chunks, chunk = task % p.chunks;
    pdl_launch_dependents();
    // (read from the parameters lane by lane, each lane another address, these would be serial for every warp)
    if (threadIdx.x < p.rot / 2) s_turns[threadIdx.x] = p.turns[threadIdx.x];
    __syncthreads();
    pdl_wait();
    if (row >= p.M) return;
    // passes of q, k and v one after another; this warp's share of them
    const int nq = (p.q.heads + HPP - 1) / HPP, nk = (p.k.heads + HPP - 1) / HPP, nv = (p.v.heads + HPP - 1) / HPP;
    const int n0 = (nq + nk + nv) * chunk / p.chunks, n1 = (nq + nk + nv) * (chunk + 1) / p.chunks;
    // loads of the passes from n on, of n's set
    auto load = [&](int n, uint4 (&x)[kInFlight]) {
        const bool is_q = n < nq, is_k = !is_q && n < nq + nk;
        const RowSet &s = is_q ? p.q : is_k ? p.k : p.v;
        const int i0 = is_q ? n : is_k ? n - nq : n - nq - nk;
        const __half *in = s.in + (long long)row * s.in_stride + 8 * l;
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            const int h = (i0 + i) * HPP + sub;
            x[i] = n + i < n1 && h < s.heads ? load_row(in + h * D) : make_uint4(0, 0, 0, 0);
        }
    };
    uint4 ahead[kInFlight];  // the first heads are on their way while the angles are computed
    load(n0, ahead);

    int pos = 0, page = 0;
    if (p.pos) pos = p.pos[row];
    if (p.cache.table) {
        const int seq = p.seq[row];
        if (seq < 0) return;  // padding
        bool ok = seq < p.cache.n_seqs && pos >= 0 && pos < kv_reach(p.cache);
        if (ok) {
            page = p.cache.table[(long long)seq * p.cache.table_stride + (pos >> p.cache.page_shift)];
            ok = kv_page_ok(p.cache, page);
        }
        if (!ok) {
            if (lane == 0) report_error(p.status, DEV_ERR_CACHE);
            return;
        }
    }
    if (p.rot > 0) {
        for (int j = lane; j < p.rot / 2; j += 32) {
            const double u = (double)pos * s_turns[j];
            float sn, cs;
            sincospif(2.0f * (float)(u - rint(u)), &sn, &cs);
            s_cos[warp][j] = cs;
            s_sin[warp][j] = sn;
        }
        __syncwarp();
    }
    const int half = p.rot / 2;
    const bool turned = 8 * l < p.rot, first = 8 * l < half;
    const int src = p.adjacent || !turned ? lane : first ? lane + half / 8 : lane - half / 8;  // who holds the pairs' other values

    auto address = [&](const RowSet &s, int h, uint16_t *pages) {
        return pages ? pages + kv_row(p.cache, page, h, pos & ((1 << p.cache.page_shift) - 1)) + 8 * l
                     : reinterpret_cast<uint16_t *>(s.out) + (long long)row * s.out_stride + h * D + 8 * l;
    };
    // passes [from, to) of a set whose first pass is pass `base` of the row
    auto turn = [&](const RowSet &s, int base, int from, int to, uint16_t *pages) {
        if (from >= to) return;
        float2 A[4], B[4];
        {
            uint4 ga = make_uint4(0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u), gb = ga;  // ones
            if (s.gamma) {
                ga = *reinterpret_cast<const uint4 *>(s.gamma + 8 * l);
                gb = *reinterpret_cast<const uint4 *>(s.gamma + 8 * (src % LPH));
            }
            const uint32_t aw[4] = {ga.x, ga.y, ga.z, ga.w}, bw[4] = {gb.x, gb.y, gb.z, gb.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                A[e] = h2_to_f2(aw[e]);
                B[e] = h2_to_f2(p.adjacent ? __byte_perm(bw[e], 0, 0x1032) : bw[e]);
                if (!turned) continue;
                if (p.adjacent) {
                    const float c = s_cos[warp][4 * l + e], sn = s_sin[warp][4 * l + e];
                    A[e] = mul2(A[e], make_float2(c, c));
                    B[e] = mul2(B[e], make_float2(-sn, sn));
                } else {
                    const int j = (first ? 8 * l : 8 * l - half) + 2 * e;
                    const float2 sn = *reinterpret_cast<const float2 *>(&s_sin[warp][j]);
                    A[e] = mul2(A[e], *reinterpret_cast<const float2 *>(&s_cos[warp][j]));
                    B[e] = mul2(B[e], first ? make_float2(-sn.x, -sn.y) : sn);
                }
            }
        }
        for (int i0 = from; i0 < to; i0 += kInFlight) {
            uint4 x[kInFlight];
#pragma unroll
            for (int i = 0; i < kInFlight; ++i) x[i] = ahead[i];
            const int next = base + min(i0 + kInFlight, to);
            if (next < n1) load(next, ahead);
#pragma unroll
            for (int i = 0; i < kInFlight; ++i) {
                if (i0 + i >= to) break;
                const int h = (i0 + i) * HPP + sub;
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                float2 y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = h2_to_f2(w[e]);
                float inv = 1.0f;
                if (s.gamma) {
                    float2 s2 = mul2(y[0], y[0]);
#pragma unroll
                    for (int e = 1; e < 4; ++e) s2 = fma2(y[e], y[e], s2);
                    float ss = s2.x + s2.y;
#pragma unroll
                    for (int d = 1; d < LPH; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
                    inv = rsqrtf(ss * (1.0f / D) + p.eps);
                }
                const float2 inv2 = make_float2(inv, inv);
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float2 r = mul2(y[e], A[e]);
                    if (p.rot > 0) {
                        const float2 z = h2_to_f2(p.adjacent ? __byte_perm(w[e], 0, 0x1032) : __shfl_sync(0xffffffffu, w[e], src));
                        // values past the rotation have no partner: an infinity must not meet a factor of 0
                        const float2 both = fma2(z, B[e], r);
                        r.x = turned ? both.x : r.x;
                        r.y = turned ? both.y : r.y;
                    }
                    r = mul2(r, inv2);
                    o[e] = f2_to_h2(r.x, r.y);
                }
                if (h < s.heads) *reinterpret_cast<uint4 *>(address(s, h, pages)) = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
    };
    turn(p.q, 0, n0, min(n1, nq), nullptr);
    turn(p.k, nq, max(n0 - nq, 0), min(n1 - nq, nk), p.cache.table ? p.cache.k : nullptr);
    for (int n = max(n0, nq + nk); n < n1; n += kInFlight) {  // values as they are
        uint4 x[kInFlight];
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) x[i] = ahead[i];
        if (n + kInFlight < n1) load(n + kInFlight, ahead);
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            const int h = (n - nq - nk + i) * HPP + sub;
            if (n + i < n1 && h < p.v.heads) *reinterpret_cast<uint4 *>(address(p.v, h, p.cache.v)) = x[i];
        }
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
    constexpr int HPP = 32 / (D / 8);
    const int passes = (p.q.heads + HPP - 1) / HPP + (p.k.heads + HPP - 1) / HPP + (p.v.heads + HPP - 1) / HPP;
    // a warp per row when the rows alone fill the GPU, else chunks of a row's passes
    p.M = M;
    p.chunks = kCtasPerSm * (kThreads / 32) * num_sms / M;
    if (p.chunks > passes) p.chunks = passes;
    if (p.chunks < 1) p.chunks = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(((long long)M * p.chunks + kThreads / 32 - 1) / (kThreads / 32)));
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
