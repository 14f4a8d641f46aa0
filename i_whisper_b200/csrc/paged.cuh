// paged.cuh -- launchers of the paged, tree-drafted decoding kernels
// (paged_plan.cu, tree_attn.cu) and of the token scores (logprobs.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace iw {

struct PlanArgs {
    const int32_t *ctx, *fresh;  // [B] cached and new tokens of each request
    int B;
    int32_t *table;
    int64_t table_ld;
    int width;
    const int32_t *free_pages;
    int64_t n_free;
    const int32_t *free_head;
    int page_log2;
    int64_t max_tokens;
    const int32_t *parents;
    int64_t max_new;
    int words;  // tree mask words per row
    int64_t *slots;
    int32_t *request, *position, *mask, *starts, *free_head_out, *status;
};
cudaError_t paged_plan(const PlanArgs &a, cudaStream_t st);

struct KvWriteArgs {
    const int8_t *k, *v;
    int64_t ldk, k_hs, ldv, v_hs;
    const int64_t *slots;
    int8_t *k_cache, *v_cache;
    int64_t page_stride, head_stride, row_stride, n_slots;
    int page_log2, H, D;
    int64_t N;
};
cudaError_t paged_kv_write(const KvWriteArgs &a, cudaStream_t st);

struct TreeAttnArgs {
    const int8_t *q;
    int64_t ldq, q_hs;
    int8_t *y;
    int64_t ldy;
    const int8_t *k, *v;
    int64_t head_stride;
    uint32_t page_stride, row_stride, n_pages;
    int page_log2;
    const int32_t *table;
    int64_t table_ld;
    int width;
    const int32_t *ctx, *starts, *mask;
    int words;  // tree mask words per row (0: chains)
    int B, H, Hkv, G, D;  // G = H / Hkv
    int64_t N;
    int32_t qk_mult;
    uint32_t qk_shift;
    int32_t frac_bits;
    int32_t av_mult;
    uint32_t av_shift, rsqrt_offset;
    bool largest_first;  // at most 32 requests, taken by decreasing work
};
cudaError_t tree_attention(const TreeAttnArgs &a, cudaStream_t st);

struct LogprobsArgs {
    const void *x;
    int64_t ld, N;
    int dtype, V;
    float scale;
    const uint32_t *suppress;
    const int64_t *targets;
    int64_t C;
    int top;
    float *lp, *entropy;
    int64_t *top_ids;
    float *top_lp;
};
cudaError_t token_logprobs(const LogprobsArgs &a, cudaStream_t st);

}  // namespace iw
