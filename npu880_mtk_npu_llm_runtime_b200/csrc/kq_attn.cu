// kq_attn.cu -- attention over the paged cache, one warp per row and head.
#include "kq_attn_dev.cuh"

namespace kq {

namespace {

constexpr int kThreads = 256;

template <int D>
__global__ __launch_bounds__(kThreads) void kq_attn_rows(const __grid_constant__ AttnLaunch p) {
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
    pdl_launch_dependents();
    pdl_wait();
    if (item >= (long long)p.M * p.heads) return;
    const int row = (int)(item / p.heads), head = (int)(item % p.heads);
    bool bad = false;
    int seq = row, pos = 0, len = 0;
    if (p.q_start) {
        for (seq = 0; seq < p.cache.n_seqs; ++seq) {
            const KvRows r = kv_rows(p.q_start[seq], p.q_start[seq + 1], p.M, bad);
            if (row >= r.begin && row < r.begin + r.n) {
                len = kv_length(p.cache, p.kv_len[seq], bad);
                pos = len - r.n + row - r.begin;
                break;
            }
        }
        if (bad && lane == 0) report_error(p.status, DEV_ERR_CACHE);
        if (seq == p.cache.n_seqs) return;  // a row of no sequence
    } else {
        len = kv_length(p.cache, p.kv_len[seq], bad);
        pos = len - 1;
        if (bad && lane == 0) report_error(p.status, DEV_ERR_CACHE);
    }
    attn_row<D>(p.cache, seq, head / (p.heads / p.cache.kv_heads), kv_span(pos, len, p.window, p.sinks),
                p.q + row * p.q_stride + head * D, p.out + row * p.out_stride + head * D, p.scale, lane, p.status);
}

template <int D>
cudaError_t launch_rows(const AttnLaunch &L, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(((long long)L.M * L.heads + kThreads / 32 - 1) / (kThreads / 32)));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = L.pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kq_attn_rows<D>, L);
}

}  // namespace

cudaError_t launch_attn_rows(const AttnLaunch &L, cudaStream_t stream) {
    switch (L.cache.head_dim) {
        case 64: return launch_rows<64>(L, stream);
        case 128: return launch_rows<128>(L, stream);
        case 256: return launch_rows<256>(L, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace kq
