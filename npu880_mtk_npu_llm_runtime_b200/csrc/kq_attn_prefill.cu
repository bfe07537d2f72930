// kq_attn_prefill.cu -- attention of ragged prompt rows over the paged cache on the 5th-generation
// tensor cores (tcgen05.mma kind::f16, accumulators in TMEM).
//
// out = sum_j w_j v_j / sum_j w_j,  w_j = 2^(x_j - m),  x_j = scale log2(e) q.k_j: one pass over
// the keys with a running maximum.  m may lag behind the true maximum by up to kLag (any m gives
// the same quotient), so the accumulated rows are rescaled only when it falls further behind.
//
// Rows: the query heads that share a key head are packed side by side, row = token * G + head, so a
// 128-row MMA tile holds 128 / G tokens and short prompts fill it too.  A CTA takes NT = 2 such
// tiles (heads of 64 and 128; 1 for 256) over the same key blocks: while the softmax of one tile
// runs, the tensor core works for the other.  Bound by the tensor pipe and the exponentials alike
// (128 x 128 x 2 x 128 operations and 128 x 128 exponentials take about the same time).  A share of the
// exponentials by polynomial on the FMA pipe made it slower (a quarter: 294 us against 289): the issue
// slots and, in long runs, the power are as scarce.
//
// Warps 0-3 and 4-7: softmax of tile 0 and 1, one row a thread: S from TMEM to registers, maximum,
// exponentials, P as fp16 back into S's columns (the second product's A operand) in two halves, and the
// epilogue.  Warp 8 issues the MMAs: P(j-1) V(j-1) then Q K(j) per tile, so S's columns are free when
// they are written.  Warps 9 and 10 load K and V page by page (TMA, 128-byte swizzle) into rings of
// blocks of BN keys, warp 9 also Q, as one box of [tokens][G heads][64 values] per 64 values; V stays as
// it lies in the cache and is the MMA's MN-major B operand.
//
// Work: an item is a row tile of one key head, a unit one of its key blocks.  Items go whole to
// the CTAs, longest first in snake order, when that balances; else (few items, long caches) every
// CTA takes an equal range of units, and the parts of an item that several CTAs share are joined
// in order by the last of them (in two steps where they are many), no finer than the joins pay for
// (make_plan).
//
// 512 rows behind 32,256 keys, 32 / 8 heads of 128: 279-295 us from run to run, 920-980 TFLOP/s, at the power cap
// (1.47 GHz); tensor pipe and exponential unit 60% busy.  A 2,048-token prompt: 42-45 us, of which 3.3 pass before
// the first block and 2.5 in each item's epilogue; a block takes 1.75 us at 1.9 GHz, 0.6 of it MMAs that the
// tile's own softmax waits for.
#include "kq_attn_dev.cuh"
#include "kq_tcgen05.cuh"

#include <cuda.h>
#include <mutex>
#include <type_traits>

namespace kq {

namespace {

// The weights are rounded to fp16, the type of the values, for the second product (fp32 sums).  They reach
// 2^(kBias + kLag), as much as fp16 holds: the rounding is half a step (2^-11) down to 2^-21 of the row's largest
// weight, and 2^-32 of it below.
constexpr float kBias = 7.0f;
constexpr float kLag = 8.0f;
// The weights' exponents are one multiply-add from the scores, x scale - m in a single rounding, but m is a
// rounded product itself: past 2^20 it is more than 1/16 off, from 2^28 on by more than fp16 holds.  Rows whose
// maximum was ever larger are computed again key by key, where score and maximum are the same product.
constexpr float kCoarse = 1048576.0f;
constexpr int kThreads = 384;  // 8 softmax warps, MMA, K and Q loads, V loads, one idle
constexpr int kWarpMma = 8, kWarpK = 9, kWarpV = 10;
constexpr int kSortTiles = 512;
// Both sides of the plan's choices are counted in blocks.  A block takes about as long for every head size: 512
// rows behind 32,256 keys give 1.8, 2.7 (at the power cap; 1.75 else) and 1.7 us a block of a CTA for heads of 64, 128
// and 256 (whose blocks are half as many keys).
// What splitting an item costs beside the blocks, its last part's wait for the others and the join, is about this
// many of them: whole items unless the fullest CTA gets that much more than an even share.
constexpr int kJoinBlocks = 8;
// What one part more costs, when the number of parts is chosen: R D / 54,000 + 0.17 blocks for R rows (256 rows of
// 128: 0.78, or 1.4 us, where the join reads such a part in 1.5 to 2).
constexpr float kPartValues = 54000.0f, kPartLatency = 0.17f;
constexpr int kJoinAhead = 3;  // parts whose values a join has on their way at once
// Parts are joined in two steps where there are more than kOneStep and together more than kOneStepRows rows (18
// parts of 128 rows 68 us against 59, of 256 rows 74 against 63; but 18 of 32 rows 45.4 against 46.9, 12 of
// 32 rows 23.4 against 25.6, 7 of 256 rows 40 against 49).
constexpr int kOneStep = 8, kOneStepRows = 1024;

template <int D>
struct Cfg {
    static constexpr int NT = D == 256 ? 1 : 2;    // MMA tiles of 128 rows
    static constexpr int BN = D == 256 ? 64 : 128; // keys of a block
    static constexpr int CH = D / 64;              // 128-byte wide pieces of a row
    static constexpr uint32_t Q_TILE = 128 * D * 2;
    static constexpr uint32_t STAGE = BN * D * 2;
    static constexpr int MAX_STAGES = 4;  // of K, and of V
    static constexpr int SOFTMAX_WARPS = 4 * NT;
    static constexpr uint32_t S_COL = BN;          // TMEM columns: S slots, then O
    static constexpr uint32_t O_COL = 256;
    static constexpr uint32_t IDESC_S = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((128u >> 4) << 24);
    static constexpr uint32_t IDESC_O = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
};

struct PrefillParams {
    AttnLaunch a;
    float scale_log2;
    int group, tpt;   // query heads of a key head; tokens of an MMA tile
    int box_rows;     // keys of one K/V box: the smaller of a page and a block
    int k_stages, v_stages;
    unsigned long long timeout_ns;
    int inject;       // 1: every CTA stops early; 2: those of odd index, so that the others' arrivals stay behind
    int wide;         // rows of out start at multiples of 32 bytes
};

// ------------------------------------------------------------------ PTX

// Shared-memory operand, 128-byte swizzle, 8-row groups 1,024 bytes apart (descriptor version 1): the
// low word (address and leading stride in 16-byte units), to which offsets in 16-byte units add, and
// the constant high word.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return ((saddr >> 4) & 0x3FFFu) | (lbo >> 4) << 16; }
constexpr uint32_t kDescHi = (1024 >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %6};\n\tmov.b64 b, {%2, %6};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(0), "r"(kDescHi));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %6};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(0), "r"(kDescHi));
}
__device__ __forceinline__ void tma4(uint32_t dst, const CUtensorMap *m, int x, int y, int z, int w, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(m), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma3(uint32_t dst, const CUtensorMap *m, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(m), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// ------------------------------------------------------------------ work

// What the CTA's roles walk: the same segments (an item, or a range of its blocks) in the same order.
struct Plan {
    const int *seq_tiles;            // [n_seqs + 1] first row tile of each sequence
    const unsigned short *order;     // whole items: row tiles, longest first (nullptr: last first)
    int tiles;                       // row tiles of all sequences
    int whole;                       // items go whole
    Shares shares;                   // else: the CTAs' shares of the units
    int start_tile;                  // else: the tile of this CTA's first unit, and that tile's first unit
    long long start_begin, c0, c1;
};

struct Segment {
    int seq, head, tile;
    int tok, n_tok;         // tokens of the sequence: first, number of them in the tile
    int row0;               // row of the first
    int pos0, len;          // its position; keys of the sequence
    KvBlocks blocks;
    KvSpan first, last;     // keys that the first and the last token see
    int b0, b1, nb;         // blocks of this segment, blocks of the item
    int live, bad;          // 0: no more segments; 1: a page that a token sees is missing
    long long begin;        // first unit of the item
};

// The row tile `tile` of sequence `seq` as a segment of all its blocks.  At least one block, so that
// a tile that sees nothing still writes its zeros.
template <int D>
__device__ __forceinline__ void tile_of(const PrefillParams &p, int seq, int tile_in_seq, Segment &s) {
    using C = Cfg<D>;
    bool bad = false;
    const KvRows rows = kv_rows(p.a.q_start[seq], p.a.q_start[seq + 1], p.a.M, bad);
    s.seq = seq;
    s.len = kv_length(p.a.cache, p.a.kv_len[seq], bad);
    s.tok = tile_in_seq * C::NT * p.tpt;
    s.n_tok = min(C::NT * p.tpt, rows.n - s.tok);
    s.row0 = rows.begin + s.tok;
    s.pos0 = s.len - rows.n + s.tok;
    s.first = kv_span(s.pos0, s.len, p.a.window, p.a.sinks);
    s.last = kv_span(s.pos0 + s.n_tok - 1, s.len, p.a.window, p.a.sinks);
    s.blocks = kv_blocks(s.last.kept, s.first.lo, s.last.hi, C::BN);
    if (s.blocks.count == 0) s.blocks.count = 1;
    s.nb = s.blocks.count;
    s.b0 = 0;
    s.b1 = s.nb;
}

__device__ __forceinline__ int seq_of_tile(const int *seq_tiles, int n_seqs, int tile) {
    int lo = 0, hi = n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (seq_tiles[mid] <= tile) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Does any token of the tile see a key of [j, j + n)?
__device__ __forceinline__ bool tile_sees(const Segment &s, int j, int n) {
    return (j < s.last.hi && j + n > s.first.lo) || j < s.last.kept;
}

template <int D>
struct Walk {
    const PrefillParams &p;
    const Plan &plan;
    unsigned k = 0;       // whole items: the CTA's next
    long long unit;       // else: the next unit
    int tile;
    long long begin;
    __device__ Walk(const PrefillParams &pp, const Plan &pl)
        : p(pp), plan(pl), unit(pl.c0), tile(pl.start_tile), begin(pl.start_begin) {}
    __device__ bool next(Segment &s) {
        const unsigned heads = p.a.cache.kv_heads;
        if (plan.whole) {
            const unsigned G = gridDim.x, c = blockIdx.x, items = plan.tiles * heads;
            unsigned idx;
            do {
                if (k * G >= items) return false;
                idx = k * G + ((k & 1) ? G - 1 - c : c);
                ++k;
            } while (idx >= items);
            const unsigned rank = idx / heads;
            s.head = (int)(idx - rank * heads);
            s.tile = plan.order ? plan.order[rank] : plan.tiles - 1 - (int)rank;
            const int seq = seq_of_tile(plan.seq_tiles, p.a.cache.n_seqs, s.tile);
            tile_of<D>(p, seq, s.tile - plan.seq_tiles[seq], s);
            s.begin = 0;
            return true;
        }
        if (unit >= plan.c1) return false;
        const int seq = seq_of_tile(plan.seq_tiles, p.a.cache.n_seqs, tile);
        tile_of<D>(p, seq, tile - plan.seq_tiles[seq], s);
        s.tile = tile;
        const unsigned r = (unsigned)(unit - begin);  // below blocks x heads of a tile: 2^24 x 2^8 at most
        s.head = (int)(r / (unsigned)s.nb);
        s.b0 = (int)(r - (unsigned)s.head * (unsigned)s.nb);
        s.begin = begin + (long long)s.head * s.nb;
        const long long left = plan.c1 - unit;
        s.b1 = s.nb - s.b0 < left ? s.nb : s.b0 + (int)left;
        unit += s.b1 - s.b0;
        if (unit >= begin + (long long)s.nb * heads) {
            begin += (long long)s.nb * heads;
            ++tile;
        }
        return true;
    }
};

// ------------------------------------------------------------------ kernel

constexpr int kSegs = 4;  // segments on their way from the loader to the other roles

struct Shared {
    unsigned long long k_full[4], k_empty[4], v_full[4], v_empty[4], q_full, q_empty, s_full[2], p_ready[2][2], o_full[2];
    unsigned long long pv_done, tail, join, never, seg_full[kSegs], seg_empty[kSegs];
    Segment seg[kSegs];
    uint32_t tmem;
    uint32_t odd[8];  // rows of each softmax warp to be mended after a join
    int abort, last, mending;  // mending: warps that compute rows key by key, which may take long
    Plan plan;
};

static_assert(sizeof(Shared) <= 1024, "a CTA has 227 KB of shared memory");
constexpr size_t kSmem = 226 * 1024;  // dynamic

// What the plan is made with, in the ring's memory.
struct PlanScratch {
    long long red[kThreads / 32], ends[kThreads / 32];
    int red_max[kThreads / 32];
    float red_split[kThreads / 32];
    int rank[kSortTiles];  // of every row tile, the longest first
    int nbs[1];            // blocks of every row tile
};

// Place in the ring: advanced block by block (a division by the number of stages would cost more than
// the rest of an MMA's issue).
struct Cursor {
    uint32_t stage = 0, phase = 0;
    __device__ __forceinline__ void next(int stages) {
        if (++stage == (uint32_t)stages) {
            stage = 0;
            phase ^= 1;
        }
    }
};

// Bounded wait on a phase: false when it did not complete in time or another role gave up.
struct Waiter {
    Shared &sh;
    unsigned long long timeout_ns;
    int *status;
    __device__ __forceinline__ bool operator()(unsigned long long &bar, uint32_t parity) const {
        const uint32_t b = smem_u32(&bar);
        if (mbar_try_wait(b, parity)) return true;
        uint64_t t0 = 0;
        for (uint32_t polls = 1;; ++polls) {
            if (mbar_try_wait(b, parity)) return true;
            if (polls & 63) continue;
            if (*reinterpret_cast<volatile int *>(&sh.abort)) return false;
            const uint64_t now = global_timer_ns();
            if (t0 == 0 || *reinterpret_cast<volatile int *>(&sh.mending)) t0 = now;
            if (now - t0 > timeout_ns) {
                *reinterpret_cast<volatile int *>(&sh.abort) = 1;
                report_error(status, DEV_ERR_TIMEOUT);
                return false;
            }
        }
    }
};

// Sum over a warp of values below 2^43 (each half of it stays below 2^32).
__device__ __forceinline__ long long sum_of_warp(long long v) {
    const unsigned lo = __reduce_add_sync(0xffffffffu, (unsigned)(v & 0xffff));
    return ((long long)__reduce_add_sync(0xffffffffu, (unsigned)(v >> 16)) << 16) + lo;
}

// The row tiles of this thread's sequences, without the ranges that begin in front of an earlier one's end, and in
// `run` their sum over the warp's lanes up to this one; by all threads.  (A call of its own: inlined, a path that no
// right call takes cost the others 2% where items are short, 700 sequences of 100 keys 143 us against 139.)
__device__ __noinline__ int disjoint_tiles(const PrefillParams &p, int *seq_tiles, int *warp_end, int s0, int chunk, int per, int &run) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, S = p.a.cache.n_seqs;
    auto row_range = [&](int s, int limit) {
        bool bad = false;
        return kv_rows_behind(p.a.q_start[s], p.a.q_start[s + 1], p.a.M, limit, bad);
    };
    int end = 0;
    for (int s = s0; s < s0 + chunk && s < S; ++s) {
        const KvRows r = row_range(s, 0);
        end = max(end, r.begin + r.n);
    }
#pragma unroll 1
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, end, d);
        if (lane >= d) end = max(end, o);
    }
    if (lane == 31) warp_end[warp] = end;
    __syncthreads();
    int limit = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) limit = 0;
    for (int w = 0; w < warp; ++w) limit = max(limit, warp_end[w]);
    int sum = 0;
    for (int s = s0; s < s0 + chunk && s < S; ++s) {
        seq_tiles[s] = sum;
        sum += (row_range(s, limit).n + per - 1) / per;
        const KvRows r = row_range(s, 0);
        limit = max(limit, r.begin + r.n);
    }
    run = sum;
#pragma unroll 1
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, run, d);
        if (lane >= d) run += o;
    }
    return sum;
}

// The CTA's plan, by all its threads (complete after the next barrier).  Every CTA makes its own: 2.4 us for one
// prompt, 1.0 of it the lengths on their way; a launch before this one would take longer.
template <int D>
__device__ __forceinline__ void make_plan(const PrefillParams &p, Shared &sh, int *seq_tiles, unsigned short *order, PlanScratch &scratch) {
    using C = Cfg<D>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, S = p.a.cache.n_seqs;
    const int per = C::NT * p.tpt;
    int *nbs = scratch.nbs;
    {
        const int chunk = (S + kThreads - 1) / kThreads, s0 = tid * chunk;
        int sum = 0;
        bool broken = false;
        for (int s = s0; s < s0 + chunk && s < S; ++s) {
            bool bad = false;
            const KvRows r = kv_rows(p.a.q_start[s], p.a.q_start[s + 1], p.a.M, bad);
            broken |= bad;
            kv_length(p.a.cache, p.a.kv_len[s], bad);
            if (bad && blockIdx.x == 0) report_error(p.a.status, DEV_ERR_CACHE);
            seq_tiles[s] = sum;
            sum += (r.n + per - 1) / per;
        }
        int run = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, run, d);
            if (lane >= d) run += o;
        }
        if (lane == 31) scratch.red[warp] = run;
        if (__syncthreads_or(broken)) {
            // q_start falls somewhere: what is valid for itself may overlap, and the tiles may then be more than the
            // tables hold.
            sum = disjoint_tiles(p, seq_tiles, scratch.red_max, s0, chunk, per, run);
            if (lane == 31) scratch.red[warp] = run;
            __syncthreads();
        }
        const int base = run - sum + __reduce_add_sync(0xffffffffu, lane < warp ? (int)scratch.red[lane] : 0);
        for (int s = s0; s < s0 + chunk && s < S; ++s) seq_tiles[s] += base;
        if (tid == kThreads - 1) seq_tiles[S] = base + sum;
        __syncthreads();
    }
    const int tiles = seq_tiles[S], heads = p.a.cache.kv_heads;
    const int chunk = (tiles + kThreads - 1) / kThreads, i0 = tid * chunk;
    long long sum = 0;
    int most = 0;
    float split = 0.0f;
    for (int i = i0; i < i0 + chunk && i < tiles; ++i) {
        Segment s;
        const int seq = seq_of_tile(seq_tiles, S, i);
        tile_of<D>(p, seq, i - seq_tiles[seq], s);
        nbs[i] = s.nb;
        sum += s.nb;
        most = max(most, s.nb);
        // an item's blocks times what joining a part of it costs, in blocks: its rows' bytes and a latency
        split = fmaxf(split, s.nb * (s.n_tok * p.group * (D / kPartValues) + kPartLatency));
    }
    {
        const long long warp_sum = sum_of_warp(sum);
        most = __reduce_max_sync(0xffffffffu, most);
        split = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(split)));  // (positive: ordered like its bits)
        if (lane == 0) {
            scratch.red[warp] = warp_sum;
            scratch.red_max[warp] = most;
            scratch.red_split[warp] = split;
        }
        if (tid < kSortTiles - kThreads) scratch.rank[kThreads + tid] = 0;
        scratch.rank[tid] = 0;
    }
    __syncthreads();
    const bool a_warp = lane < kThreads / 32;  // each warp puts the warps' values together
    const long long total = sum_of_warp(a_warp ? scratch.red[lane] : 0) * heads;
    most = __reduce_max_sync(0xffffffffu, a_warp ? scratch.red_max[lane] : 0);
    split = __uint_as_float(__reduce_max_sync(0xffffffffu, a_warp ? __float_as_uint(scratch.red_split[lane]) : 0u));
    // Whole items in snake order, unless the fullest CTA would get more than an even share and a join.
    const int G = gridDim.x, items = tiles * heads;
    const Shares even(total > 0 ? total : 1, G);
    // Without a look at the order where there are many items, short enough that no CTA can get more than twice an even
    // share (the look costs 3 us of 120 for 4,800 items of a block).  A long item among them: one sequence of 131,072
    // keys and 600 of 100 take 330 us in equal shares, whole 1,650.
    bool whole = items >= 32 * G && (long long)((items + G - 1) / G) * most <= 2 * even.q, ordered = false;
    if (!whole && most <= even.q + kJoinBlocks) {
        // longest first: from the last tile on where no tile is longer than the next (one prompt), else by rank
        bool rising = true;
        for (int i = max(i0, 1); i < i0 + chunk && i < tiles; ++i) rising &= nbs[i - 1] <= nbs[i];
        ordered = !__syncthreads_and(rising);
        if (ordered && tiles <= kSortTiles) {
            const int by = max(kThreads / tiles, 1);  // threads that share a tile's comparisons
            for (int e = tid; e < tiles * by; e += kThreads) {
                const int i = e % tiles, n = nbs[i];
                int rank = 0;
                for (int j = e / tiles; j < tiles; j += by) rank += nbs[j] > n || (nbs[j] == n && j < i);
                atomicAdd(&scratch.rank[i], rank);
            }
            __syncthreads();
            for (int i = tid; i < tiles; i += kThreads) order[scratch.rank[i]] = (unsigned short)i;
            __syncthreads();
        }
        int fits = !ordered || tiles <= kSortTiles;
        for (int c = tid; fits && c < G; c += kThreads) {
            int sum = 0;
            for (int k = 0; k * G < items; ++k) {
                const int idx = k * G + ((k & 1) ? G - 1 - c : c), rank = (unsigned)idx / (unsigned)heads;
                if (idx < items) sum += nbs[ordered ? order[rank] : tiles - 1 - rank];
            }
            fits = sum <= even.q + kJoinBlocks;
        }
        whole = __syncthreads_and(fits);
    }
    Plan &pl = sh.plan;
    if (tid == 0) {
        pl.seq_tiles = seq_tiles;
        pl.order = ordered ? order : nullptr;
        pl.tiles = tiles;
        pl.whole = whole;
    }
    if (whole) {
        if (tid == 0) {
            pl.start_tile = 0;
            pl.start_begin = pl.c0 = pl.c1 = 0;
        }
        return;
    }
    // Split: shares of x blocks take x and joining an item of n blocks (n / x) c blocks' time, least at
    // x = sqrt(n c); more CTAs than that would spend longer joining than they save.
    const int parts = (int)fmaxf(fminf((float)G, (float)total * rsqrtf(fmaxf(split, 1.0f))), 1.0f);
    const Shares shares = parts == G ? even : Shares(total > 0 ? total : 1, parts);
    long long run = sum;
#pragma unroll 1
    for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, run, d);
        if (lane >= d) run += o;
    }
    if (lane == 31) scratch.ends[warp] = run;
    const bool mine = total > 0 && (int)blockIdx.x < parts;
    const long long c0 = mine ? shares.begin(blockIdx.x) : 0, c1 = mine ? shares.begin(blockIdx.x + 1) : 0;
    if (tid == 0) {
        pl.shares = shares;
        pl.c0 = c0;
        pl.c1 = c1;
        if (c1 <= c0) {
            pl.start_tile = 0;
            pl.start_begin = 0;
        }
    }
    __syncthreads();
    if (c1 > c0) {  // (uniform over the CTA)
        long long before = run - sum + sum_of_warp(lane < warp ? scratch.ends[lane] : 0);
        for (int i = i0; i < i0 + chunk && i < tiles; ++i) {
            if (before * heads <= c0 && c0 < (before + nbs[i]) * heads) {
                pl.start_tile = i;
                pl.start_begin = before * heads;
            }
            before += nbs[i];
        }
    }
}

// Loads of one CTA by a warp each: the K warp hands the segments to the other roles and loads Q and K,
// the V warp loads V (two warps, because a block of 16-position pages is 16 copies or more, which one warp
// issues no faster than the MMAs read it).  `at`: the ring's next block.
template <int D, bool V>
__device__ __forceinline__ void load_role(const PrefillParams &p, Shared &sh, const Waiter &wait, const CUtensorMap &mq,
                                          const CUtensorMap &m, unsigned char *s_q, unsigned char *s_ring, int lane, Cursor &at) {
    using C = Cfg<D>;
    constexpr int NT = C::NT, BN = C::BN, CH = C::CH;
    const AttnLaunch &a = p.a;
    const int boxes = (BN / p.box_rows) * CH, stages = V ? p.v_stages : p.k_stages;
    const int sub = lane / CH, piece = lane % CH;  // this lane's box of a block
    uint32_t tails = 0;
    Walk<D> walk(p, sh.plan);
    for (uint32_t k = 0;; ++k) {
        Segment s;
        Segment &rec = sh.seg[k % kSegs];
        if (V) {
            if (!wait(sh.seg_full[k % kSegs], (k / kSegs) & 1)) return;
            s = rec;
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.seg_empty[k % kSegs]));
        } else {
            const bool have = walk.next(s);
            if (!wait(sh.seg_empty[k % kSegs], ((k / kSegs) & 1) ^ 1)) return;
            s.bad = 0;
            s.live = have;
            if (lane == 0) {
                rec = s;
                mbar_arrive(smem_u32(&sh.seg_full[k % kSegs]));
            }
            __syncwarp();
        }
        if (!s.live) return;
        const int32_t *table = a.cache.table + (long long)s.seq * a.cache.table_stride;
        // This lane's box of block i in the table: read a block ahead, looked at when it is needed.
        struct Entry {
            int page;
            bool sees;  // whether any token sees the box
        };
        auto entry_of = [&](int i) {
            const int j = kv_block(s.blocks, i) * BN + sub * p.box_rows;
            Entry e{0, lane < boxes && i < s.b1 && tile_sees(s, j, p.box_rows)};
            if (e.sees) e.page = table[j >> a.cache.page_shift];
            return e;
        };
        auto load_q = [&] {
            const int subs = s.n_tok > p.tpt ? NT : 1;
            if (!wait(sh.q_empty, (k & 1) ^ 1)) return false;
            if (lane == 0) mbar_arrive_expect_tx(smem_u32(&sh.q_full), (uint32_t)(subs * p.tpt * p.group * D * 2));
            __syncwarp();
            if (lane < subs * CH)
                tma3(smem_u32(s_q) + sub * C::Q_TILE + piece * (128 * 128), &mq, 64 * piece, s.head * p.group,
                     s.row0 + sub * p.tpt, smem_u32(&sh.q_full));
            __syncwarp();
            return true;
        };
        Entry here = entry_of(s.b0);
        if (!V && k == 0 && !load_q()) return;  // (later items' queries wait for room: not before their first keys)
        for (int i = s.b0; i < s.b1; ++i) {
            const Entry next = entry_of(i + 1);
            const uint32_t st = at.stage;
            if (!wait((V ? sh.v_empty : sh.k_empty)[st], at.phase ^ 1)) return;
            at.next(stages);
            const int j0 = kv_block(s.blocks, i) * BN;
            unsigned char *to = s_ring + (size_t)st * C::STAGE;
            unsigned long long &full = (V ? sh.v_full : sh.k_full)[st];
            // V rows past the sequence's end may hold anything, and 0 * NaN is NaN: zeroed once they landed
            const bool tail = V && j0 + BN > s.len;
            const uint32_t bar = smem_u32(tail ? &sh.tail : &full);
            // a box that no token sees, or whose page is missing: n_pages, out of range, is filled with zeros
            const bool ok = here.sees && kv_page_ok(a.cache, here.page);
            if (!V && here.sees && !ok) *reinterpret_cast<volatile int *>(&rec.bad) = 1;
            const int page = ok ? here.page : a.cache.n_pages;
            __syncwarp();
            if (lane == 0) mbar_arrive_expect_tx(bar, C::STAGE);
            __syncwarp();
            if (lane < boxes)
                tma4(smem_u32(to) + piece * (BN * 128) + sub * p.box_rows * 128, &m, 64 * piece,
                     (j0 + sub * p.box_rows) & ((1 << a.cache.page_shift) - 1), s.head, page, bar);
            if (tail) {
                if (!wait(sh.tail, tails & 1)) return;
                ++tails;
                for (int e = lane + max(0, s.len - j0) * 8; e < BN * 8; e += 32)
#pragma unroll
                    for (int c = 0; c < CH; ++c)
                        *reinterpret_cast<uint4 *>(to + c * (BN * 128) + e * 16) = make_uint4(0, 0, 0, 0);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&full));
            }
            __syncwarp();
            here = next;
            if (!V && k > 0 && i == s.b0 && !load_q()) return;
        }
    }
}

// After an early stop: let a warp's copies in flight land before the CTA's memory goes (bounded).
__device__ __forceinline__ void drain(unsigned long long *full, int stages, const Cursor &at) {
    const uint64_t t0 = global_timer_ns();
    for (uint32_t i = 0; i < (uint32_t)stages; ++i)  // (a stage not yet used this time round completed before)
        while (!mbar_test_wait(smem_u32(full + i), at.phase ^ (i >= at.stage)) && global_timer_ns() - t0 < 2000000ull) {
        }
    while (global_timer_ns() - t0 < 50000ull) {
    }
}

// The MMAs of one CTA, by a converged warp, one elected lane issuing.
template <int D>
__device__ __forceinline__ void mma_role(const PrefillParams &p, Shared &sh, const Waiter &wait, uint32_t q0, uint32_t k_ring,
                                         uint32_t v_ring, uint32_t tmem) {
    using C = Cfg<D>;
    constexpr int NT = C::NT, BN = C::BN;
    constexpr uint32_t kStep = C::STAGE >> 4;
    Cursor ka, va;            // the rings' next blocks to read
    uint32_t np[2] = {0, 0};  // P's begun of each slot
    if (p.inject && (p.inject == 1 || (blockIdx.x & 1)) && !wait(sh.never, 0)) return;
    const uint32_t q_lo = desc_lo(q0, 16), k_lo = desc_lo(k_ring, 16), v_lo = desc_lo(v_ring, BN * 128);
    // S slot = Q tile t times the K block in ring stage st
    auto mma_s = [&](int t, int slot, uint32_t st) {
        const uint32_t kb = k_lo + st * kStep, qb = q_lo + t * (C::Q_TILE >> 4);
#pragma unroll
        for (int e = 0; e < D / 16; ++e)
            mma_ss(tmem + slot * C::S_COL, qb + (e / 4) * (128 * 128 / 16) + (e % 4) * 2, kb + (e / 4) * (BN * 128 / 16) + (e % 4) * 2,
                   C::IDESC_S, e > 0);
        tc_commit(smem_u32(&sh.s_full[slot]));
    };
    // O tile t (+)= half h of the slot's P times its keys' rows of the V block in ring stage st
    auto mma_o = [&](int t, int slot, uint32_t st, bool first, int h) {
        const uint32_t vb = v_lo + st * kStep + h * (BN / 32) * 128, pb = tmem + slot * C::S_COL + h * (BN / 4);
#pragma unroll
        for (int e = 0; e < BN / 32; ++e)
            mma_ts(tmem + C::O_COL + t * D, pb + e * 8, vb + e * 128, C::IDESC_O, !(first && h == 0 && e == 0));
    };
    // a half of the slot's next P (each half has a barrier of its own: both may come before either is waited for)
    auto wait_p = [&](int slot, int h) { return wait(sh.p_ready[slot][h], (h == 0 ? np[slot]++ : np[slot] - 1) & 1); };
    for (uint32_t k = 0;; ++k) {
        if (!wait(sh.seg_full[k % kSegs], (k / kSegs) & 1)) return;
        const Segment &s = sh.seg[k % kSegs];
        if (!s.live) return;
        const int subs = s.n_tok > p.tpt ? NT : 1, nb = s.b1 - s.b0;
        __syncwarp();
        if (elect_one()) mbar_arrive(smem_u32(&sh.seg_empty[k % kSegs]));
        if (!wait(sh.q_full, k & 1)) return;
        for (int j = -(3 - NT); j < nb; ++j) {
            // PV of block j, S of block j + 3 - NT (a tile a slot: the next; one tile: the next but one, whose slot
            // is free then)
            const int js = j + 3 - NT;
            const uint32_t v = va.stage, kk = ka.stage;
            if (j >= 0) {
                if (!wait(sh.v_full[v], va.phase)) return;
                va.next(p.v_stages);
            }
            if (js < nb) {
                if (!wait(sh.k_full[kk], ka.phase)) return;
                ka.next(p.k_stages);
            }
            for (int t = 0; t < subs; ++t) {
                const int slot = NT == 2 ? t : j & 1;
                if (j >= 0) {
                    if (!wait_p(slot, 0)) return;
                    tc_fence_after();
                    if (elect_one()) mma_o(t, slot, v, j == 0, 0);
                    __syncwarp();
                    if (!wait_p(slot, 1)) return;
                }
                tc_fence_after();
                if (elect_one()) {
                    if (j >= 0) {
                        mma_o(t, slot, v, false, 1);
                        if (j == nb - 1) tc_commit(smem_u32(&sh.o_full[t]));
                        else if (NT == 1) tc_commit(smem_u32(&sh.pv_done));
                        if (t == subs - 1) tc_commit(smem_u32(&sh.v_empty[v]));
                    }
                    if (js < nb) {
                        mma_s(t, slot, kk);
                        if (t == subs - 1) {
                            tc_commit(smem_u32(&sh.k_empty[kk]));
                            if (js == nb - 1) tc_commit(smem_u32(&sh.q_empty));
                        }
                    }
                }
                __syncwarp();
            }
        }
    }
}

// Rows of a warp whose plain result does not stand: computed key by key, over exactly their own
// keys.  These see nothing (zeros), or have a value that is not finite: a weight of 0 times an
// infinity that only other rows see is NaN in the matrix product; or a page is missing; or their scores
// are too large (kCoarse).  (Another row whose sum is NaN saw a NaN score: all NaN, which stands.)
template <int D>
__device__ __forceinline__ void mend_rows(const PrefillParams &p, Shared &sh, const Segment &s, bool odd, int tok, int head,
                                          int lane) {
    uint32_t todo = __ballot_sync(0xffffffffu, odd);
    if (!todo) return;
    __syncwarp();  // the rows' plain results, stored by a lane each, before other lanes store over them (votes order no memory)
    if (lane == 0) atomicAdd(&sh.mending, 1);
    while (todo) {
        const int src = __ffs(todo) - 1;
        todo &= todo - 1;
        const int tk = __shfl_sync(0xffffffffu, tok, src), hd = __shfl_sync(0xffffffffu, head, src);
        const long long row = s.row0 + tk;
        attn_row<D>(p.a.cache, s.seq, s.head, kv_span(s.pos0 + tk, s.len, p.a.window, p.a.sinks),
                    p.a.q + row * p.a.q_stride + hd * D, p.a.out + row * p.a.out_stride + hd * D, p.a.scale, lane, p.a.status);
    }
    __syncwarp();
    if (lane == 0) atomicSub(&sh.mending, 1);
}

// 32 values of a row, times `by`, rounded, to out (where `write`).  `odd` turns NaN when one is not
// finite (0 times it is NaN); such a row is computed again, so its infinities need not be kept here.
// With rows that allow it 32 bytes a store: a warp's lanes write to 32 rows, so a 16-byte store would
// fill half a sector at each.
__device__ __forceinline__ void put32(const float *o, float by, uint16_t *out, bool write, bool wide, float2 &odd) {
    uint32_t h[16];
    const float2 by2 = make_float2(by, by), zero = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const float2 v = __fmul2_rn(make_float2(o[2 * e], o[2 * e + 1]), by2);
        odd = __ffma2_rn(v, zero, odd);
        h[e] = finite_mean_to_h2(v.x, v.y);
    }
    if (!write) return;
    if (wide) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(out + 16 * e), "r"(h[8 * e]), "r"(h[8 * e + 1]),
                         "r"(h[8 * e + 2]), "r"(h[8 * e + 3]), "r"(h[8 * e + 4]), "r"(h[8 * e + 5]), "r"(h[8 * e + 6]), "r"(h[8 * e + 7])
                         : "memory");
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint4 *>(out + 8 * e) = make_uint4(h[4 * e], h[4 * e + 1], h[4 * e + 2], h[4 * e + 3]);
    }
}

// Softmax and epilogue of row tile t, by 128 threads with a row each.
template <int D>
__device__ __forceinline__ void softmax_role(const PrefillParams &p, Shared &sh, const Waiter &wait, uint32_t tmem) {
    using C = Cfg<D>;
    constexpr int NT = C::NT, BN = C::BN;
    constexpr int part_rows = NT * 128;
    const AttnLaunch &a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t = warp >> 2, r = tid & 127;
    const uint32_t lane_base = tmem + ((uint32_t)(warp & 3) << 21);
    const uint32_t o_base = lane_base + C::O_COL + t * D;
    uint32_t ns[2] = {0, 0}, no = 0, npv = 0, nj = 0;
    // all softmax warps of the CTA (bounded, unlike a hardware barrier)
    auto together = [&] {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.join));
        return wait(sh.join, nj++ & 1);
    };
    for (uint32_t k = 0;; ++k) {
        if (!wait(sh.seg_full[k % kSegs], (k / kSegs) & 1)) return;
        const Segment &s = sh.seg[k % kSegs];
        if (!s.live) return;
        const bool active = t == 0 || s.n_tok > p.tpt;
        const bool whole = s.b0 == 0 && s.b1 == s.nb;
        const int tok = t * p.tpt + r / p.group, head = s.head * p.group + r % p.group;
        const bool mine = active && r < p.tpt * p.group && tok < s.n_tok;
        uint16_t *out = a.out + (long long)(s.row0 + tok) * a.out_stride + head * D;
        if (active) {
            const KvSpan span = kv_span(s.pos0 + tok, s.len, a.window, a.sinks);
            // blocks in [all_lo, all_hi) or below all_kept: every row of the tile sees them whole
            const int all_hi = kv_span(s.pos0 + t * p.tpt, s.len, a.window, a.sinks).hi;
            const int all_kept = kv_span(s.pos0 + t * p.tpt, s.len, a.window, a.sinks).kept;
            const int all_lo = kv_span(s.pos0 + min(s.n_tok, (t + 1) * p.tpt) - 1, s.len, a.window, a.sinks).lo;
            const int b0 = s.b0, b1 = s.b1;
            const KvBlocks blocks = s.blocks;
            float m = -INFINITY, l = 0.0f;
            bool coarse = false;  // see kCoarse
            for (int i = b0; i < b1; ++i) {
                const int slot = NT == 2 ? t : (i - b0) & 1;
                const uint32_t s_base = lane_base + slot * C::S_COL;
                const int j0 = kv_block(blocks, i) * BN;
                const bool full = j0 + BN <= all_hi && (j0 >= all_lo || j0 + BN <= all_kept);
                if (!wait(sh.s_full[slot], ns[slot] & 1)) return;
                ++ns[slot];
                tc_fence_after();
                float x[BN];
#pragma unroll
                for (int c = 0; c < BN / 32; ++c) tmem_ld32(s_base + 32 * c, reinterpret_cast<uint32_t *>(x + 32 * c));
                tmem_wait_ld();
                if (!full) {
#pragma unroll
                    for (int c = 0; c < BN / 32; ++c) {
                        // bit e: the row sees key j0 + 32 c + e
                        auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
                        const int at = j0 + 32 * c;
                        const uint32_t bits = below(span.hi - at) & (~below(span.lo - at) | below(span.kept - at));
#pragma unroll
                        for (int e = 0; e < 32; ++e) x[32 * c + e] = (bits >> e & 1) ? x[32 * c + e] : -INFINITY;
                    }
                }
                float mx[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) mx[u] = fmaxf(x[2 * u], x[2 * u + 1]);
#pragma unroll
                for (int e = 8; e < BN; e += 8)
#pragma unroll
                    for (int u = 0; u < 4; ++u) mx[u] = max3(mx[u], x[e + 2 * u], x[e + 2 * u + 1]);
                const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * p.scale_log2;
                const bool raise = top > m + kLag;  // the first score above -inf raises from -inf
                if (__any_sync(0xffffffffu, raise)) {
                    const float to = raise ? top : m;
                    coarse |= raise && fabsf(top) > kCoarse;
                    const float alpha = m == to ? 1.0f : exp2_fast(m - to);
                    l *= alpha;
                    m = to;
                    if (i > b0) {
                        if (NT == 1) {
                            // S of this block only tells that P V of the block before the last is done
                            if (!wait(sh.pv_done, (npv + (i - b0) - 1) & 1)) return;
                            tc_fence_after();
                        }
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            tmem_ld16(o_base + 16 * c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                            tmem_st16(o_base + 16 * c, o);
                        }
                    }
                }
                const float off = (m == -INFINITY ? 0.0f : -m) + kBias;
                const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), off2 = make_float2(off, off);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int half = 0; half < 2; ++half) {  // P goes to the MMA in halves: the first runs while the second is made
#pragma unroll
                    for (int c = half * (BN / 64); c < (half + 1) * (BN / 64); ++c) {
                        uint32_t h[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float2 w = __ffma2_rn(make_float2(x[32 * c + 2 * e], x[32 * c + 2 * e + 1]), scale2, off2);
                            w.x = exp2_fast(w.x);
                            w.y = exp2_fast(w.y);
                            sum[e & 1] = __fadd2_rn(sum[e & 1], w);
                            h[e] = f2_to_h2(w.x, w.y);
                        }
                        tmem_st16(s_base + 16 * c, h);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sh.p_ready[slot][half]));
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            if (!wait(sh.o_full[t], no & 1)) return;
            ++no;
            npv += b1 - b0 - 1;
            tc_fence_after();
            const bool bad = *reinterpret_cast<const volatile int *>(&s.bad) != 0;
            if (whole) {
                float2 odd = make_float2(0.0f, 0.0f);
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    float o[32];
                    tmem_ld32(o_base + 32 * c, reinterpret_cast<uint32_t *>(o));
                    tmem_wait_ld();
                    put32(o, 1.0f / l, out + 32 * c, mine, p.wide, odd);
                }
                mend_rows<D>(p, sh, s, mine && (bad || coarse || m == -INFINITY || (l == l && !(odd.x + odd.y == 0.0f))), tok, head, lane);
            } else {
                // this CTA's part: [value / 4][row][4], then (m, l) of each row
                float4 *part = reinterpret_cast<float4 *>(a.parts + (size_t)(2 * blockIdx.x + (b0 == 0)) * part_rows * (D + 2)) + t * 128 + r;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    float o[32];
                    tmem_ld32(o_base + 32 * c, reinterpret_cast<uint32_t *>(o));
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (mine) part[(8 * c + e) * part_rows] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                }
                reinterpret_cast<float2 *>(part - (t * 128 + r) + D / 4 * part_rows)[t * 128 + r] = make_float2(bad || coarse ? NAN : m, l);  // NaN: to be computed again
            }
        }
        if (!whole) {
            // The last CTA that brings a part of the item joins them in order; or, in two steps, the last of every
            // `fan` CTAs joins theirs (in place of the first one's part) and the last of all what comes of that: a
            // CTA reads a part of 256 rows in 1.5-2 us, and so has fan + n / fan of them on its way, not n.
            const int first = sh.plan.shares.of(s.begin);
            const int last = sh.plan.shares.of(s.begin + s.nb - 1), n = last - first + 1;
            // A tile of 32 or 64 rows gives its other warps shares of the values.
            const int rows = active ? min(s.n_tok - t * p.tpt, p.tpt) * p.group : 0;
            const int span_warps = rows <= 32 ? 1 : rows <= 64 ? 2 : 4, shares = 4 / span_warps;
            const int jr = (warp & (span_warps - 1)) * 32 + lane;  // this thread's row of the tile
            const bool on = jr < rows;
            auto part_at = [&](int c) { return reinterpret_cast<float4 *>(a.parts + (size_t)(2 * c + (c == first)) * part_rows * (D + 2)); };
            auto stat_at = [&](int c) { return reinterpret_cast<float2 *>(part_at(c) + D / 4 * part_rows) + t * 128 + jr; };
            // whether this CTA is the last of `others` + 1
            auto arrive = [&](unsigned *count, int others, bool &join) {
                if (!together()) return false;
                if (tid == 0) {
                    // after the barrier: the release covers all of the CTA's rows
                    sh.last = count_arrival(count) == (unsigned)others;
                    if (sh.last) *count = 0;  // for the next launch
                }
                if (!together()) return false;
                join = sh.last != 0;
                return together();
            };
            // The parts of CTAs from, from + step, .. to: 32 values of a row at a time to put(c0, o); the row's statistics.
            auto join_parts = [&](int from, int to, auto step, float &M, float &L, bool &missing, auto put) {
                M = -INFINITY;
                L = 0.0f;
                missing = false;
                if (!on) return;
#pragma unroll 8
                for (int c = from; c <= to; c += step) {
                    const float2 ml = __ldcg(stat_at(c));
                    missing |= ml.x != ml.x;
                    const float top = fmaxf(M, ml.x);
                    // a part without a score above -inf adds nothing; NaN (a NaN score) stays
                    L = L * (M == -INFINITY ? 1.0f : exp2_fast(M - top)) +
                        (ml.x == -INFINITY ? (ml.y != ml.y ? ml.y : 0.0f) : exp2_fast(ml.x - top) * ml.y);
                    M = top;
                }
                for (int c0 = 32 * ((warp & 3) / span_warps); c0 < D; c0 += 32 * shares) {
                    float o[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0.0f;
#pragma unroll 1
                    for (int c = from; c <= to; c += kJoinAhead * step) {
                        float4 v[kJoinAhead][8];
                        float w[kJoinAhead];
#pragma unroll
                        for (int i = 0; i < kJoinAhead; ++i) {
                            const int cc = min(c + i * step, to);
                            const float4 *part = part_at(cc) + c0 / 4 * part_rows + t * 128 + jr;
                            w[i] = __ldcg(stat_at(cc)).x;
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[i][e] = __ldcg(part + e * part_rows);
                        }
#pragma unroll
                        for (int i = 0; i < kJoinAhead; ++i) {
                            if (c + i * step > to) break;
                            w[i] = w[i] == -INFINITY ? 0.0f : exp2_fast(w[i] - M);
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                o[4 * e] += w[i] * v[i][e].x;
                                o[4 * e + 1] += w[i] * v[i][e].y;
                                o[4 * e + 2] += w[i] * v[i][e].z;
                                o[4 * e + 3] += w[i] * v[i][e].w;
                            }
                        }
                    }
                    put(c0, o, L);
                }
            };
            float M, L;
            bool missing, join;
            float2 odd = make_float2(0.0f, 0.0f);
            const int jtok = t * p.tpt + jr / p.group, jhead = s.head * p.group + jr % p.group;
            uint16_t *jout = a.out + (long long)(s.row0 + jtok) * a.out_stride + jhead * D;
            auto result = [&](int c0, const float *o, float l) { put32(o, 1.0f / l, jout + c0, true, p.wide, odd); };
            const std::integral_constant<int, 1> one;
            if (n <= kOneStep || n * s.n_tok * p.group <= kOneStepRows) {
                if (!arrive(a.count + first, n - 1, join)) return;
                if (join) join_parts(first, last, one, M, L, missing, result);
            } else {
                const int fan = (int)ceilf(sqrtf((float)n)), g = ((int)blockIdx.x - first) / fan;
                const int from = first + g * fan, to = min(from + fan - 1, last);
                if (!arrive(a.count + (int)gridDim.x + 2 * from + (g == 0), to - from, join)) return;
                if (join) {
                    join_parts(from, to, 1, M, L, missing, [&](int c0, const float *o, float) {  // (nobody else reads these)
                        float4 *part = part_at(from) + c0 / 4 * part_rows + t * 128 + jr;
#pragma unroll
                        for (int e = 0; e < 8; ++e) part[e * part_rows] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    });
                    if (!together()) return;  // the row's other threads have read its old statistics
                    if (on && (warp & 3) < span_warps) *stat_at(from) = make_float2(missing ? NAN : M, L);
                    if (!arrive(a.count + first, (n - 1) / fan, join)) return;
                    if (join) join_parts(first, first + (n - 1) / fan * fan, fan, M, L, missing, result);
                }
            }
            if (join) {
                __syncwarp();
                const uint32_t wrong = __ballot_sync(0xffffffffu, on && (missing || M == -INFINITY || (L == L && !(odd.x + odd.y == 0.0f))));
                if (lane == 0 && wrong) atomicOr(&sh.odd[t * 4 + (warp & (span_warps - 1))], wrong);
                if (!together()) return;  // all values are written
                const uint32_t mend = sh.odd[warp];
                __syncwarp();
                if (lane == 0) sh.odd[warp] = 0;  // (every warp has read its own before the next join's first meeting)
                mend_rows<D>(p, sh, s, mend >> lane & 1, tok, head, lane);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.seg_empty[k % kSegs]));
    }
}

template <int D>
__global__ __launch_bounds__(kThreads, 1) void kq_attn_prefill(const __grid_constant__ PrefillParams p,
                                                               const __grid_constant__ CUtensorMap mq,
                                                               const __grid_constant__ CUtensorMap mk,
                                                               const __grid_constant__ CUtensorMap mv) {
    using C = Cfg<D>;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ Shared sh;
    const AttnLaunch &a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned char *s_q = smem, *s_k = smem + C::NT * C::Q_TILE, *s_v = s_k + (size_t)p.k_stages * C::STAGE;
    int *seq_tiles = reinterpret_cast<int *>(s_v + (size_t)p.v_stages * C::STAGE);
    unsigned short *order = reinterpret_cast<unsigned short *>(seq_tiles + a.cache.n_seqs + 1);

    pdl_launch_dependents();
    if (tid == 32) {
        for (const CUtensorMap *m : {&mq, &mk, &mv}) asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    }
    if (tid == 0) {
        auto init = [](unsigned long long &bar, uint32_t count) { mbar_init(smem_u32(&bar), count); };
        for (int i = 0; i < C::MAX_STAGES; ++i) {
            init(sh.k_full[i], 1);
            init(sh.k_empty[i], 1);
            init(sh.v_full[i], 1);
            init(sh.v_empty[i], 1);
        }
        init(sh.q_full, 1);
        init(sh.q_empty, 1);
        for (int t = 0; t < 2; ++t) {
            init(sh.s_full[t], 1);
            init(sh.p_ready[t][0], 4);
            init(sh.p_ready[t][1], 4);
            init(sh.o_full[t], 1);
        }
        init(sh.pv_done, 1);
        init(sh.tail, 1);
        init(sh.join, C::SOFTMAX_WARPS);
        init(sh.never, 1);
        for (int i = 0; i < kSegs; ++i) {
            init(sh.seg_full[i], 1);
            init(sh.seg_empty[i], C::SOFTMAX_WARPS + 2);
        }
        mbar_init_fence();
        sh.abort = 0;
        sh.mending = 0;
        for (int i = 0; i < 8; ++i) sh.odd[i] = 0;
    }
    if (warp == kWarpMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    pdl_wait();
    make_plan<D>(p, sh, seq_tiles, order, *reinterpret_cast<PlanScratch *>(s_k));
    fence_async_smem();  // the ring's memory goes from the plan to the TMA
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const Waiter wait{sh, p.timeout_ns, a.status};

    if (warp >= kWarpMma) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == kWarpK) {
            Cursor at;
            load_role<D, false>(p, sh, wait, mq, mk, s_q, s_k, lane, at);
            __syncwarp();
            if (*reinterpret_cast<volatile int *>(&sh.abort)) drain(sh.k_full, p.k_stages, at);
        } else if (warp == kWarpV) {
            Cursor at;
            load_role<D, true>(p, sh, wait, mq, mv, s_q, s_v, lane, at);
            __syncwarp();
            if (*reinterpret_cast<volatile int *>(&sh.abort)) drain(sh.v_full, p.v_stages, at);
        } else if (warp == kWarpMma) {
            mma_role<D>(p, sh, wait, smem_u32(s_q), smem_u32(s_k), smem_u32(s_v), tmem);
            __syncwarp();
            if (*reinterpret_cast<volatile int *>(&sh.abort)) {
                // let the MMAs in flight end before the accumulators go (bounded)
                if (elect_one()) tc_commit(smem_u32(&sh.never));
                __syncwarp();
                const uint64_t t0 = global_timer_ns();
                while (!mbar_test_wait(smem_u32(&sh.never), 0) && global_timer_ns() - t0 < 2000000ull) {
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        if (warp < C::SOFTMAX_WARPS) softmax_role<D>(p, sh, wait, tmem);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kWarpMma) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// ------------------------------------------------------------------ host

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
    static EncodeFn fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult r{};
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeFn>(f);
    }();
    return fn;
}

bool encode(CUtensorMap *m, const void *base, int rank, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box) {
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    return encode_fn()(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank, const_cast<void *>(base), dims, strides, box, ones,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
cudaError_t launch(PrefillParams &p, cudaStream_t stream) {
    using C = Cfg<D>;
    const AttnLaunch &a = p.a;
    const int page = 1 << a.cache.page_shift;
    p.box_rows = page < C::BN ? page : C::BN;
    // most row tiles: one per sequence more than the rows fill
    const size_t tables = (size_t)(a.cache.n_seqs + 1) * 4 + (size_t)kSortTiles * 2;
    const size_t room = kSmem - tables - C::NT * C::Q_TILE;
    const int stages = (int)(room / C::STAGE);  // K, which is waited for longest, gets the odd one
    p.k_stages = (stages + 1) / 2 < C::MAX_STAGES ? (stages + 1) / 2 : C::MAX_STAGES;
    p.v_stages = stages / 2 < C::MAX_STAGES ? stages / 2 : C::MAX_STAGES;
    const size_t smem = C::NT * C::Q_TILE + (size_t)(p.k_stages + p.v_stages) * C::STAGE + tables;

    CUtensorMap mq, mk, mv;
    const cuuint64_t qd[3] = {(cuuint64_t)D, (cuuint64_t)a.heads, (cuuint64_t)a.M};
    const cuuint64_t qs[2] = {(cuuint64_t)D * 2, (cuuint64_t)a.q_stride * 2};
    const cuuint32_t qb[3] = {64, (cuuint32_t)p.group, (cuuint32_t)p.tpt};
    const cuuint64_t kd[4] = {(cuuint64_t)D, (cuuint64_t)page, (cuuint64_t)a.cache.kv_heads, (cuuint64_t)a.cache.n_pages};
    const cuuint64_t ks[3] = {(cuuint64_t)D * 2, (cuuint64_t)page * D * 2, (cuuint64_t)page * D * 2 * a.cache.kv_heads};
    const cuuint32_t kb[4] = {64, (cuuint32_t)p.box_rows, 1, 1};
    if (!encode_fn()) return cudaErrorNotSupported;
    if (!encode(&mq, a.q, 3, qd, qs, qb) || !encode(&mk, a.cache.k, 4, kd, ks, kb) || !encode(&mv, a.cache.v, 4, kd, ks, kb))
        return cudaErrorInvalidValue;
    {
        static std::mutex mu;
        static bool configured[64] = {};
        int dev = 0;
        cudaGetDevice(&dev);
        std::lock_guard<std::mutex> lk(mu);
        if (dev < 0 || dev >= 64 || !configured[dev]) {
            cudaError_t e = cudaFuncSetAttribute(kq_attn_prefill<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)kSmem);
            if (e != cudaSuccess) return e;
            if (dev >= 0 && dev < 64) configured[dev] = true;
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.num_sms);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = a.pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kq_attn_prefill<D>, p, mq, mk, mv);
}

}  // namespace

size_t attn_prefill_part_bytes(int num_sms) {
    size_t most = 0;
    for (size_t rows_d : {(size_t)256 * (64 + 2), (size_t)256 * (128 + 2), (size_t)128 * (256 + 2)})
        if (rows_d > most) most = rows_d;
    return (size_t)2 * num_sms * most * 4;
}

cudaError_t launch_attn_prefill(const AttnLaunch &L, cudaStream_t stream) {
    PrefillParams p{};
    p.a = L;
    p.scale_log2 = L.scale * 1.4426950408889634f;
    p.group = L.heads / L.cache.kv_heads;
    p.tpt = 128 / p.group;
    p.timeout_ns = L.timeout_ns;
    p.inject = L.inject;
    p.wide = kv_aligned(L.out, 32) && L.out_stride % 16 == 0;
    switch (L.cache.head_dim) {
        case 64: return launch<64>(p, stream);
        case 128: return launch<128>(p, stream);
        case 256: return launch<256>(p, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace kq
