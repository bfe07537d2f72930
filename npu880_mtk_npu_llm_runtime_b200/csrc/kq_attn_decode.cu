// kq_attn_decode.cu -- attention of one new token per sequence over the paged cache.
//
// out = sum_j w_j v_j / sum_j w_j,  w_j = 2^(x_j - m),  x_j = scale log2(e) q.k_j,  m a running
// maximum: one pass over K and V.  Two parts (m, l = sum w, o = sum w v) of one row join as
// M = max(m, m'), l 2^(m - M) + l' 2^(m' - M), and o likewise.
//
// Bound by the cache's bytes: every visible key and value once, 4 D bytes for 4 D G operations
// (G query heads share a key head; of heads of 256 the registers hold 8 at a time, so with more of them a key head is
// two items, and its bytes come twice: see below).  So the work is cut by bytes: a unit is 16 keys of one
// (sequence, key head) item, the units of all items stand in one row, and every CTA (one per SM)
// and in it every warp takes an equal, contiguous range of them -- few or many sequences, equal
// or ragged, load the SMs alike.  A warp works alone, without shared memory or barriers, and keeps
// a whole unit (16 keys, 4 KB of K and 4 KB of V at D = 128) in flight in registers; the parts
// of an item that several warps share meet in shared memory, those that several CTAs share in
// global memory, joined in unit order by the last CTA that arrives (many parts in two steps: one
// sequence of 14,000 keys, 16 query heads on one key head, 21 us where one step takes 77).
//
// The products run on mma.m16n8k16 with the keys (then the values' dimensions) as the 16 rows and
// the query heads as the 8 columns, so a group of up to 8 heads wastes nothing of the registers:
//   S^T = K Q^T: a lane's 16-byte load of a key row is its A fragment of two steps, because which
//   k slot stands for which dimension is free as long as Q's B fragment uses the same order;
//   O^T = V^T P^T: lane (g, t) loads dimensions 8g.. of keys 2t, 2t+1, 2t+8, 2t+9 and pairs the
//   keys of a dimension with byte permutes; P^T's fragment is S^T's transposed by movmatrix.
// tcgen05 has nothing to add here: the tensor pipe (8.7% busy) idles either way while the bytes come in.
//
// 4 sequences x 131,072 keys, 8 key heads of 128 (2.15 GB): 327-346 us from run to run, 6.2-6.5 TB/s, 0.95-0.99 of a
// measured copy; 64 sequences of 1..8,192 keys (239 MB): 49 us, of which 38 stream; 1 x 1,000 keys: 10 us, six dependent
// memory latencies and the launch.  16 x 8,192 keys read 1.0004 x their bytes from DRAM.
// Heads of 256, 4 key heads, 65,536 keys (268 MB): 57 us with 4 query heads a key head, 62 with 8 (4.4 TB/s; 8 warps an SM,
// 255 registers and 68 bytes of spills), 83 with 16: the two items of a key head are read at the same time, so DRAM gives 1.01 x the
// bytes and L2 the second copy.
#include "kq_attn_dev.cuh"

#include <mutex>
#include <type_traits>

namespace kq {

namespace {

// The weights are rounded to fp16, the type of the values, for the second product; all sums, that of the weights
// too, stay fp32 (32-bit weights would need a second product of their low parts).  They reach 2^kBias, as much as
// fp16 holds: the rounding is half a step (2^-11) down to 2^-29 of the largest weight, and 2^-40 of it below.
constexpr float kBias = 15.0f;
constexpr float kLeastHalf = 5.9604645e-8f;  // fp16's smallest number: weights for the second product, as kLeast
constexpr int kUnit = 16;  // keys of a unit; a page holds a multiple of it
// Beginning an item (its queries, its first page) costs a warp about as much as this many units:
// every item counts that many more when the work is cut, or the warps with the short sequences
// would end last.
constexpr int kBegin = 2;
constexpr int kJoin = 3;
constexpr int kFan = 12;  // parts that a thread joins one after another (148: two steps of 12)
constexpr int kAhead = 6;  // of them on their way at once, ..
constexpr int kFew = 3;    // .. but where there are no more than this one by one (less code to fetch)

template <int D, int NB>
struct Cfg {
    // Registers of a lane: Q D/8 NB, O D/4 NB, K and V D/4 each, so D = 256 takes 8 heads at a time; as many
    // warps as they allow, for the bytes in flight (D = 64: 16 warps 69 us where 12 take 76, 373 MB).
    static constexpr int WARPS = (D * NB == 64) ? 16 : (D * NB <= 128) ? 12 : 8;
    static constexpr int THREADS = 32 * WARPS;
};

struct DecodeParams {
    AttnLaunch a;
    float scale_log2;
    int group, rows, splits;  // query heads of a key head; of an item; items of a key head
    int part_floats;          // floats of a part: rows x (D + 2), to a multiple of 16 bytes
    int floats;               // shared memory before the tables
    float *parts;             // [2][CTA][2] parts (and joined ones) of rows x D values, then [rows][2] (m, l)
    unsigned *count;          // [CTA] arrivals at the item that begins in a CTA and ends in a later one; then
                              // [CTA][2] at the groups of its parts
};

// The cache streams through: first to leave L2, so that what is used again (the kernel's code, the
// tables, the parts) stays there.  (Not the read-only path: the kernel may be resident before the one
// that appends the last rows has ended.)
__device__ __forceinline__ uint4 load_stream(const uint16_t *p, uint64_t policy) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.L2::cache_hint.v4.u32 {%0,%1,%2,%3}, [%4], %5;"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p), "l"(policy));
    return v;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ float max_over_keys(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float sum_over_keys(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 4);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

struct Item {
    int seq, vhead, cost;  // sequence, item of the sequence (key head x splits), kBegin + its units
    long long begin;       // where its cost begins; its first unit stands kBegin later
};

// prefix[s]: cost of one item of each of the sequences 0..s-1; `per` items a sequence
__device__ __forceinline__ Item item_of(const int *prefix, int n_seqs, int per, long long unit) {
    int lo = 0, hi = n_seqs;  // prefix[lo] * per <= unit < prefix[hi] * per
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((long long)prefix[mid] * per <= unit) lo = mid;
        else hi = mid;
    }
    Item it;
    it.seq = lo;
    it.cost = prefix[lo + 1] - prefix[lo];
    const long long first = (long long)prefix[lo] * per, r = unit - first;
    it.vhead = (int)((float)r / (float)it.cost);  // at most 2^9: one off at most
    if ((long long)it.vhead * it.cost > r) --it.vhead;
    if ((long long)(it.vhead + 1) * it.cost <= r) ++it.vhead;
    it.begin = first + (long long)it.vhead * it.cost;
    return it;
}

// Parts of a row joined one after another: four of its values.  A part with nothing above -inf is
// marked: m = -inf, and l = 0 when it saw no key, +inf when every score was -inf, NaN when one was NaN.
struct Joint {
    float M = -INFINITY, L = 0.0f;
    bool seen = false;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __device__ __forceinline__ void add(float2 ml, float4 x) {
        const float top = fmaxf(M, ml.x);
        const float old = M == -INFINITY ? 1.0f : at_least(exp2f(M - top), kLeast);  // before the first score: L is 0 or NaN, v is 0
        const float w = ml.x == -INFINITY ? 0.0f : at_least(exp2f(ml.x - top), kLeast);
        L = L * old + (ml.x == -INFINITY ? (ml.y != ml.y ? ml.y : 0.0f) : w * ml.y);
        v.x = v.x * old + w * x.x;
        v.y = v.y * old + w * x.y;
        v.z = v.z * old + w * x.z;
        v.w = v.w * old + w * x.w;
        M = top;
        seen |= ml.x > -INFINITY || ml.y > 0.0f;
    }
    __device__ __forceinline__ float2 mark() const {
        return make_float2(M, M == -INFINITY && seen && L == 0.0f ? INFINITY : L);
    }
    // scores all -inf: 0 / 0, NaN as in the formula; no key there: zeros
    __device__ __forceinline__ uint2 result() const {
        if (!seen && L == L) return make_uint2(0u, 0u);
        const float inv = 1.0f / L;
        return make_uint2(mean_to_h2(v.x * inv, v.y * inv), mean_to_h2(v.z * inv, v.w * inv));
    }
};

// A warp's part of an item: which one, where its rows go, and the item's units.
struct PartInfo {
    int id;  // -1: none
    int seq, head0, n_rows;
    long long begin, end;  // of its units
};

template <int D, int NB>
__global__ __launch_bounds__(Cfg<D, NB>::THREADS, 1) void kq_attn_decode(const __grid_constant__ DecodeParams p) {
    using C = Cfg<D, NB>;
    constexpr int KC = D / 32;  // 16-byte pieces of a key row per lane
    constexpr int VC = D / 64;  // of a value row
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int s_warp[C::WARPS];
    __shared__ PartInfo s_part[2 * C::WARPS];  // each warp's first and last part
    __shared__ uint32_t s_run[2 * C::WARPS];  // the parts of each item, as bits
    __shared__ int s_runs;                    // items that have parts
    __shared__ int s_last[2];
    const AttnLaunch &a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int S = a.cache.n_seqs, per = a.cache.kv_heads * p.splits;
    const int part_floats = p.part_floats;
    float *s_parts = reinterpret_cast<float *>(smem);
    int *prefix = reinterpret_cast<int *>(s_parts + p.floats);
    int *lens = prefix + S + 1;

    pdl_launch_dependents();
    pdl_wait();

    // units of every sequence, and where they begin
    int most = 0;
    {
        const int chunk = (S + C::THREADS - 1) / C::THREADS, s0 = tid * chunk;
        int sum = 0;
        for (int s = s0; s < s0 + chunk && s < S; ++s) {
            bool bad = false;
            const int len = kv_length(a.cache, a.kv_len[s], bad);
            lens[s] = len;
            if (bad && blockIdx.x == 0) report_error(a.status, DEV_ERR_CACHE);
            const KvSpan sp = kv_span(len - 1, len, a.window, a.sinks);
            const int n = kv_blocks(sp.kept, sp.lo, sp.hi, kUnit).count;
            prefix[s] = sum;
            sum += n ? n + kBegin : 0;
            most = max(most, n);
            if (n == 0 && s % gridDim.x == blockIdx.x)  // sees nothing: zeros
                for (int i = 0; i < a.heads * D / 8; ++i)
                    *reinterpret_cast<uint4 *>(a.out + s * a.out_stride + 8 * i) = make_uint4(0, 0, 0, 0);
        }
        int run = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, run, d);
            if (lane >= d) run += o;
        }
        if (lane == 31) s_warp[warp] = run;
        if (tid < 2 * C::WARPS) s_part[tid].id = -1;
        __syncthreads();
        int base = run - sum;
        for (int w = 0; w < warp; ++w) base += s_warp[w];
        for (int s = s0; s < s0 + chunk && s < S; ++s) prefix[s] += base;
        if (tid == C::THREADS - 1) prefix[S] = base + sum;
        __syncthreads();
    }
    const long long total = (long long)prefix[S] * per;
    // An item a CTA, with nothing to join across CTAs, where there are CTAs enough and the longest item is not
    // longer than an even share and what a join costs (kJoin units a warp); else equal shares, of no more CTAs
    // than give every warp a unit.  (1 sequence of 400 keys: 9.0 us against 9.5; 16 of 1,000: 18.9 against
    // 20.9; 1 of 1,000: 13.8 against 10.0, so split.)
    bool solo = S * per <= (int)gridDim.x;
    if (solo) solo = !__syncthreads_or(most > (int)(total / gridDim.x) + kJoin * C::WARPS);
    const int parts = solo ? S * per : (int)min((long long)gridDim.x, (total + C::WARPS - 1) / C::WARPS);
    if ((int)blockIdx.x >= parts) return;
    const Shares shares(total, parts);
    long long c0 = shares.begin(blockIdx.x), c1 = shares.begin(blockIdx.x + 1);
    if (solo) {
        const int seq = blockIdx.x / per, cost = prefix[seq + 1] - prefix[seq];
        if (cost == 0) return;
        c0 = (long long)prefix[seq] * per + (long long)(blockIdx.x % per) * cost + kBegin;
        c1 = c0 + cost - kBegin;
    }
    const Shares mine_shares(c1 - c0, C::WARPS);
    const long long w0 = c0 + mine_shares.begin(warp), w1 = c0 + mine_shares.begin(warp + 1);

    const uint64_t policy = l2_evict_first_policy();
    int slot = 0;  // this warp's next part in shared memory
    for (long long unit = w0; unit < w1;) {
        const Item it = item_of(prefix, S, per, unit);
        const int kv_head = it.vhead / p.splits, row0 = (it.vhead % p.splits) * p.rows;
        const int n_rows = min(p.rows, p.group - row0);
        const int to = (int)min((long long)it.cost, w1 - it.begin);
        const int t0 = max((int)(unit - it.begin) - kBegin, 0), t1 = max(to - kBegin, 0);
        unit = it.begin + to;
        if (t0 == t1) continue;  // nothing but the item's beginning
        const int len = lens[it.seq];
        const KvSpan span = kv_span(len - 1, len, a.window, a.sinks);
        const KvBlocks blocks = kv_blocks(span.kept, span.lo, span.hi, kUnit);
        const int head0 = kv_head * p.group + row0;
        const int32_t *table = a.cache.table + (long long)it.seq * a.cache.table_stride;

        uint4 q[NB][KC];
        float o[NB][VC * 4][4], m[NB][2], l[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int r = 8 * b + g;
#pragma unroll
            for (int c = 0; c < KC; ++c)
                q[b][c] = r < n_rows ? *reinterpret_cast<const uint4 *>(a.q + it.seq * a.q_stride + (head0 + r) * D + 32 * c + 8 * t)
                                     : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < VC * 4; ++i) o[b][i][0] = o[b][i][1] = o[b][i][2] = o[b][i][3] = 0.0f;
            m[b][0] = m[b][1] = -INFINITY;
            l[b][0] = l[b][1] = 0.0f;
        }
        bool seen = false;
        int next_page = table[(kv_block(blocks, t0) * kUnit) >> a.cache.page_shift];
        for (int i = t0; i < t1; ++i) {
            const int j0 = kv_block(blocks, i) * kUnit;
            const int page = next_page;
            if (i + 1 < t1) next_page = table[(kv_block(blocks, i + 1) * kUnit) >> a.cache.page_shift];
            if (!kv_page_ok(a.cache, page)) {  // uniform: the unit counts as masked
                if (lane == 0) report_error(a.status, DEV_ERR_CACHE);
                continue;
            }
            const long long row = kv_row(a.cache, page, kv_head, j0 & ((1 << a.cache.page_shift) - 1));
            const uint16_t *kp = a.cache.k + row + 8 * t, *vp = a.cache.v + row + 8 * g;
            // Keys that the row does not see are not loaded: zeros stand for them, whatever they hold.
            const bool full = j0 >= span.lo && j0 + kUnit <= span.hi;
            const bool k0 = full || kv_sees(span, j0 + g), k1 = full || kv_sees(span, j0 + g + 8);
            uint4 kr[2][KC], vr[4][VC];
            const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                kr[0][c] = k0 ? load_stream(kp + g * D + 32 * c, policy) : zero;
                kr[1][c] = k1 ? load_stream(kp + (g + 8) * D + 32 * c, policy) : zero;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int key = 2 * t + (u & 1) + 4 * (u & 2);
                const bool vis = full || kv_sees(span, j0 + key);
#pragma unroll
                for (int c = 0; c < VC; ++c) vr[u][c] = vis ? load_stream(vp + key * D + 64 * c, policy) : zero;
            }
            seen = true;
            uint32_t pb[NB][2];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    mma_f16(s, kr[0][c].x, kr[1][c].x, kr[0][c].y, kr[1][c].y, q[b][c].x, q[b][c].y);
                    mma_f16(s, kr[0][c].z, kr[1][c].z, kr[0][c].w, kr[1][c].w, q[b][c].z, q[b][c].w);
                }
                // s[0], s[1]: key g, rows 2t, 2t+1; s[2], s[3]: key g+8
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] = (e < 2 ? k0 : k1) ? __fmul_rn(s[e], p.scale_log2) : -INFINITY;
                float al[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float mn = fmaxf(m[b][e], max_over_keys(fmaxf(s[e], s[e + 2])));
                    const float ref = (mn == -INFINITY) ? 0.0f : mn;
                    al[e] = at_least(exp2f(m[b][e] - ref), kLeast);
                    m[b][e] = mn;
                    const float w0 = exp2f(s[e] - ref + kBias), w1 = exp2f(s[e + 2] - ref + kBias);
                    l[b][e] = l[b][e] * al[e] + (w0 + w1);
                    s[e] = s[e] == -INFINITY ? 0.0f : at_least(w0, kLeastHalf);
                    s[e + 2] = s[e + 2] == -INFINITY ? 0.0f : at_least(w1, kLeastHalf);
                }
                if (__any_sync(0xffffffffu, al[0] != 1.0f || al[1] != 1.0f)) {
#pragma unroll
                    for (int i2 = 0; i2 < VC * 4; ++i2) {
                        o[b][i2][0] *= al[0];
                        o[b][i2][1] *= al[1];
                        o[b][i2][2] *= al[0];
                        o[b][i2][3] *= al[1];
                    }
                }
                pb[b][0] = transpose8x8(f2_to_h2(s[0], s[1]));
                pb[b][1] = transpose8x8(f2_to_h2(s[2], s[3]));
            }
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    const uint32_t x0 = word(vr[0][c], jj), x1 = word(vr[1][c], jj);
                    const uint32_t x2 = word(vr[2][c], jj), x3 = word(vr[3][c], jj);
                    const uint32_t a0 = __byte_perm(x0, x1, 0x5410), a1 = __byte_perm(x0, x1, 0x7632);
                    const uint32_t a2 = __byte_perm(x2, x3, 0x5410), a3 = __byte_perm(x2, x3, 0x7632);
#pragma unroll
                    for (int b = 0; b < NB; ++b) mma_f16(o[b][4 * c + jj], a0, a1, a2, a3, pb[b][0], pb[b][1]);
                }
        }

        // o[b][4c + jj]: dimensions 64c + 8g + 2jj (elements 0, 1) and the next (2, 3), rows 2t (0, 2), 2t+1 (1, 3)
        const bool whole = t0 == 0 && t1 == it.cost - kBegin;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float sum = sum_over_keys(l[b][e]);
                const int r = 8 * b + 2 * t + e;
                if (r >= n_rows) continue;
                if (whole) {
                    // scores all -inf: 0 / 0 as in the formula; no key there: zeros
                    const float inv = seen ? 1.0f / sum : 0.0f;
#pragma unroll
                    for (int c = 0; c < VC; ++c) {
                        uint32_t v[4];
#pragma unroll
                        for (int jj = 0; jj < 4; ++jj) v[jj] = mean_to_h2(o[b][4 * c + jj][e] * inv, o[b][4 * c + jj][e + 2] * inv);
                        *reinterpret_cast<uint4 *>(a.out + it.seq * a.out_stride + (head0 + r) * D + 64 * c + 8 * g) =
                            make_uint4(v[0], v[1], v[2], v[3]);
                    }
                } else {
                    float *part = s_parts + (size_t)(2 * warp + slot) * part_floats;
#pragma unroll
                    for (int c = 0; c < VC; ++c)
#pragma unroll
                        for (int jj = 0; jj < 4; ++jj)
                            *reinterpret_cast<float2 *>(part + r * D + 64 * c + 8 * g + 2 * jj) =
                                make_float2(o[b][4 * c + jj][e], o[b][4 * c + jj][e + 2]);
                    if (g == 0) {
                        part[p.rows * D + 2 * r] = m[b][e];
                        part[p.rows * D + 2 * r + 1] = (m[b][e] == -INFINITY && seen && sum == 0.0f) ? INFINITY : sum;
                    }
                }
            }
        if (!whole) {
            if (lane == 0) s_part[2 * warp + slot] = PartInfo{it.seq * per + it.vhead, it.seq, head0, n_rows, it.begin + kBegin, it.begin + it.cost};
            ++slot;
        }
    }
    __syncthreads();

    // Join the warps' parts of each item (they stand in unit order): into the output, or into this
    // CTA's part of an item that other CTAs share too.
    if (warp == 0) {
        const int id = lane < 2 * C::WARPS ? s_part[lane].id : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, id);
        const bool lead = id >= 0 && lane == __ffs(same) - 1;
        const uint32_t leads = __ballot_sync(0xffffffffu, lead);
        if (lead) s_run[__popc(leads & ((1u << lane) - 1u))] = same;
        if (lane == 0) s_runs = __popc(leads);
    }
    __syncthreads();
    const int elems = p.rows * (D / 4);  // a thread takes four values of a row
    const int runs = s_runs;
    // the item that began before this CTA, and the one that goes on after it: their parts (-1: none)
    int before = -1, after = -1;
    if (runs > 0) {
        const int i0 = __ffs(s_run[0]) - 1, i1 = __ffs(s_run[runs - 1]) - 1;
        if (s_part[i0].begin < c0) before = i0;
        if (s_part[i1].end > c1 && s_part[i1].begin >= c0) after = i1;
    }
    for (int e = tid; e < runs * elems; e += C::THREADS) {
        uint32_t bits = s_run[e / elems];
        const int lead = __ffs(bits) - 1;
        const int r = (e % elems) / (D / 4), d = 4 * (e % (D / 4));
        const PartInfo &info = s_part[lead];
        if (r >= info.n_rows) continue;
        Joint jn;
#pragma unroll 1
        for (; bits; bits &= bits - 1) {
            const float *part = s_parts + (size_t)(__ffs(bits) - 1) * part_floats;
            jn.add(*reinterpret_cast<const float2 *>(part + p.rows * D + 2 * r), *reinterpret_cast<const float4 *>(part + r * D + d));
        }
        if (lead == before || lead == after) {
            float *part = p.parts + (size_t)(2 * blockIdx.x + (lead == before ? 0 : 1)) * part_floats;
            *reinterpret_cast<float4 *>(part + r * D + d) = jn.v;
            if (d == 0) *reinterpret_cast<float2 *>(part + p.rows * D + 2 * r) = jn.mark();
        } else {
            *reinterpret_cast<uint2 *>(a.out + info.seq * a.out_stride + (info.head0 + r) * D + d) = jn.result();
        }
    }
    if (before < 0 && after < 0) return;  // uniform over the CTA

    // Items shared with other CTAs: the last to arrive joins their parts in unit order.  Where a thread would have
    // more than kFan of them one after another, the last of every fan CTAs joins those first (into a second set of
    // parts), and the last of all what comes of that.
    const int groups = elems < C::THREADS ? C::THREADS / elems : 1;  // threads left over share the parts
    const int fan = kFan * groups, G = gridDim.x, me = blockIdx.x;
    int first[2] = {0, 0}, last[2] = {0, 0};
    if (before >= 0) {
        first[0] = shares.of(s_part[before].begin);
        last[0] = s_part[before].end > c1 ? shares.of(s_part[before].end - 1) : me;
    }
    if (after >= 0) {
        first[1] = me;
        last[1] = shares.of(s_part[after].end - 1);
    }
    const bool many[2] = {last[0] - first[0] >= kFew * groups, last[1] - first[1] >= kFew * groups};
    __syncthreads();
    if (tid < 2) {
        int is_last = 0;
        if ((tid ? after : before) >= 0) {
            const int f = tid ? first[1] : first[0], l = tid ? last[1] : last[0];
            unsigned *count = p.count + f;
            int others = l - f;
            if (others >= fan) {
                const int g0 = f + (me - f) / fan * fan;
                count = p.count + G + 2 * g0 + (g0 == f);
                others = min(fan - 1, l - g0);
            }
            // after the barrier: the release covers the whole CTA's part
            is_last = count_arrival(count) == (unsigned)others;
            if (is_last) *count = 0;  // for the next launch
        }
        s_last[tid] = is_last;
    }
    __syncthreads();
    float2 *s_ml = reinterpret_cast<float2 *>(s_parts + 4 * C::THREADS);
    float4 *s_v = reinterpret_cast<float4 *>(s_parts);
    // n parts, the i-th at part(i), `ahead` of them on their way at once; put(r, d, joint) takes every four values
    auto join = [&](auto ahead, int n_rows, int n, auto part, auto put) {
        constexpr int A = decltype(ahead)::value;
        for (int e0 = 0; e0 < elems; e0 += C::THREADS) {
            const int e = groups > 1 ? tid % elems : e0 + tid, grp = groups > 1 ? tid / elems : 0;
            const int r = e / (D / 4), d = 4 * (e % (D / 4));
            const bool on = e < elems && grp < groups && r < n_rows;
            Joint jn;
            if (on) {
#pragma unroll 1
                for (int i = grp; i < n; i += A * groups) {
                    float2 ml[A];
                    float4 v[A];
#pragma unroll
                    for (int u = 0; u < A; ++u) {
                        const float *from = part(A > 1 ? min(i + u * groups, n - 1) : i);
                        ml[u] = __ldcg(reinterpret_cast<const float2 *>(from + p.rows * D + 2 * r));
                        v[u] = __ldcg(reinterpret_cast<const float4 *>(from + r * D + d));
                    }
#pragma unroll
                    for (int u = 0; u < A; ++u)
                        if (u == 0 || i + u * groups < n) jn.add(ml[u], v[u]);
                }
                if (grp > 0) {
                    s_v[tid] = jn.v;
                    s_ml[tid] = jn.mark();
                }
            }
            if (groups > 1) __syncthreads();
            if (on && grp == 0) {
                for (int k = 1; k < groups; ++k) jn.add(s_ml[k * elems + e], s_v[k * elems + e]);
                put(r, d, jn);
            }
        }
        __syncthreads();
    };
    if (many[0] || many[1]) {
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
            if (!s_last[which] || !(which ? many[1] : many[0])) continue;  // uniform over the CTA
            const PartInfo info = s_part[which ? after : before];
            const int f = which ? first[1] : first[0], l = which ? last[1] : last[0];
            const bool two = l - f >= fan;
            int at = f, step = 1, n = l - f + 1;  // the parts of CTAs at, at + step, ..; joined ones: G further on
            float *to = nullptr;
            if (two) {
                at = f + (me - f) / fan * fan;
                n = min(fan, l - at + 1);
                to = p.parts + (size_t)(2 * (G + at) + (at == f)) * part_floats;
            }
            while (true) {
                const int begins = at == f || at == G + f;  // the first part is of the CTA where the item begins
                join(std::integral_constant<int, kAhead>(), info.n_rows, n,
                     [&](int i) { return p.parts + (size_t)(2 * (at + step * i) + (i == 0 ? begins : 0)) * part_floats; },
                     [&](int r, int d, const Joint &jn) {
                         if (to) {
                             *reinterpret_cast<float4 *>(to + r * D + d) = jn.v;
                             if (d == 0) *reinterpret_cast<float2 *>(to + p.rows * D + 2 * r) = jn.mark();
                         } else {
                             *reinterpret_cast<uint2 *>(a.out + info.seq * a.out_stride + (info.head0 + r) * D + d) = jn.result();
                         }
                     });
                if (!to) break;
                if (tid == 0) {
                    s_last[which] = count_arrival(p.count + f) == (unsigned)((l - f) / fan);
                    if (s_last[which]) p.count[f] = 0;
                }
                __syncthreads();
                if (!s_last[which]) break;
                at = G + f;
                step = fan;
                n = (l - f) / fan + 1;
                to = nullptr;
            }
        }
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (!s_last[which] || many[which]) continue;  // uniform over the CTA
        const PartInfo info = s_part[which ? after : before];
        const int f = first[which], n = last[which] - f + 1;
        join(std::integral_constant<int, 1>(), info.n_rows, n,
             [&](int i) { return p.parts + (size_t)(2 * (f + i) + (i == 0)) * part_floats; },
             [&](int r, int d, const Joint &jn) {
                 *reinterpret_cast<uint2 *>(a.out + info.seq * a.out_stride + (info.head0 + r) * D + d) = jn.result();
             });
    }
}

template <int D, int NB>
cudaError_t launch(DecodeParams &p, cudaStream_t stream) {
    using C = Cfg<D, NB>;
    p.rows = p.group < 8 * NB ? p.group : 8 * NB;
    p.splits = (p.group + p.rows - 1) / p.rows;
    // the warps' parts; later, in the same place, the threads' sums of a join
    p.part_floats = (p.rows * (D + 2) + 3) & ~3;
    const size_t room = (size_t)2 * C::WARPS * p.part_floats * 4, join = (size_t)C::THREADS * 24;
    p.floats = (int)((room > join ? room : join) / 4);
    const size_t smem = (size_t)p.floats * 4 + (size_t)(2 * p.a.cache.n_seqs + 1) * 4;
    {
        static std::mutex mu;
        static bool configured[64] = {};
        int dev = 0;
        cudaGetDevice(&dev);
        std::lock_guard<std::mutex> lk(mu);
        if (dev < 0 || dev >= 64 || !configured[dev]) {
            cudaError_t e = cudaFuncSetAttribute(kq_attn_decode<D, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
            if (e != cudaSuccess) return e;
            if (dev >= 0 && dev < 64) configured[dev] = true;
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.a.num_sms);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = p.a.pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kq_attn_decode<D, NB>, p);
}

}  // namespace

size_t attn_decode_part_bytes(int num_sms) { return (size_t)4 * num_sms * KQ_MAX_GROUP * (KQ_MAX_HEAD_DIM + 2) * 4; }

cudaError_t launch_attn_decode(const AttnLaunch &L, cudaStream_t stream) {
    DecodeParams p{};
    p.a = L;
    p.scale_log2 = L.scale * 1.4426950408889634f;
    p.group = L.heads / L.cache.kv_heads;
    p.parts = L.parts;
    p.count = L.count;
    const bool wide = p.group > 8;
    switch (L.cache.head_dim) {
        case 64: return wide ? launch<64, 2>(p, stream) : launch<64, 1>(p, stream);
        case 128: return wide ? launch<128, 2>(p, stream) : launch<128, 1>(p, stream);
        case 256: return launch<256, 1>(p, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace kq
