// kq_attn.h -- host-side launch descriptions of the attention operators.
#pragma once

#include <cuda_runtime.h>

#include "kq_kv.h"

namespace kq {

// Norms, rotation and append (kq_rope.cu).  cache == nullptr: no append, v unused.
struct RopeLaunch {
    const kq_heads *q, *k, *v;
    const KvView *cache;
    const kq_rope *rope;
    int head_dim, M;
    const int32_t *seq, *pos;
    float eps;
    int *status;
    int num_sms;
    bool pdl;
};
cudaError_t launch_norm_rope(const RopeLaunch &L, cudaStream_t stream);

// Attention over the cache: M rows, of one token per sequence (q_start == nullptr)
// or of the sequences' last rows.
struct AttnLaunch {
    KvView cache;
    const uint16_t *q;
    long long q_stride;
    uint16_t *out;
    long long out_stride;
    int heads, M;
    const int32_t *kv_len, *q_start;
    int window, sinks;
    float scale;
    int *status;
    int num_sms;
    bool pdl;
    // scratch: parts of rows that several CTAs share; arrival counts, all zero between launches
    float *parts;
    unsigned *count;
    unsigned long long timeout_ns;
    int inject;  // failure-path test hook (see kq_set_option "inject_timeout")
};
// kq_attn_prefill.cu
size_t attn_prefill_part_bytes(int num_sms);
cudaError_t launch_attn_prefill(const AttnLaunch &L, cudaStream_t stream);
// kq_attn_decode.cu
size_t attn_decode_part_bytes(int num_sms);
// arrival counts: an item's, and its two groups' (see DecodeParams)
inline size_t attn_counts(int num_sms) { return (size_t)3 * num_sms; }
cudaError_t launch_attn_decode(const AttnLaunch &L, cudaStream_t stream);
}  // namespace kq
