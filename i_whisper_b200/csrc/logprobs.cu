// logprobs.cu -- log probabilities of given tokens, entropy and the most
// likely tokens of each row of logits (iw_token_logprobs). With l = scale * x
// over the tokens that are not suppressed, m = max l and S = sum exp(l - m),
//   lp(t) = l_t - m - ln S,   H = ln S - sum (l - m) exp(l - m) / S.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "iw_common.cuh"
#include "paged.cuh"

namespace iw {

constexpr int kLpThreads = 256;

template <typename T>
IW_DEV float lp_float(T v) { return (float)v; }
template <>
IW_DEV float lp_float<__half>(__half v) { return __half2float(v); }
template <>
IW_DEV float lp_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// One block per row: maximum, sums, then one pass over the row per
// alternative. A rank (value, id) is one 64-bit key: the float's bits made
// to order as an unsigned number, then the id inverted so that the lowest wins.
IW_DEV uint64_t lp_key(float v, uint32_t id) {
    const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);
    const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((uint64_t)o << 32) | (uint32_t)~id;
}
IW_DEV float lp_key_value(uint64_t k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

template <typename F, typename T>
IW_DEV T lp_block_reduce(T v, F f, T *red) {
    __syncthreads();
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < kLpThreads / 32; ++w) v = f(v, red[w]);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(LogprobsArgs a) {
    pdl_wait();
    pdl_launch();
    __shared__ uint64_t red_k[kLpThreads / 32];
    __shared__ float red_f[kLpThreads / 32];
    const int64_t n = blockIdx.x;
    const T *x = reinterpret_cast<const T *>(a.x) + n * a.ld;
    auto gone = [&](int64_t i) { return a.suppress && ((a.suppress[i >> 5] >> (i & 31)) & 1u); };
    auto most = [](uint64_t p, uint64_t q) { return p > q ? p : q; };
    auto add = [](float p, float q) { return p + q; };
    uint64_t best = 0;
    float bad = 0.f;
    for (int i = threadIdx.x; i < a.V; i += kLpThreads) {
        if (gone(i)) continue;
        const float v = lp_float(x[i]);
        if (!(v < INFINITY)) bad = 1.f;
        else if (v > -INFINITY) best = most(best, lp_key(v, i));
    }
    bad = lp_block_reduce(bad, add, red_f);
    best = lp_block_reduce(best, most, red_k);
    const float m = best ? lp_key_value(best) * a.scale : 0.f;
    float S = 0.f, W = 0.f;
    for (int i = threadIdx.x; i < a.V; i += kLpThreads) {
        if (gone(i)) continue;
        const float d = lp_float(x[i]) * a.scale - m;
        const float e = expf(d);
        S += e;
        if (e > 0.f) W += e * d;
    }
    S = lp_block_reduce(S, add, red_f);
    W = lp_block_reduce(W, add, red_f);
    const float ln = logf(S);
    const bool is_bad = bad > 0.f, none = best == 0;
    if (threadIdx.x == 0) a.entropy[n] = is_bad ? NAN : (none ? 0.f : ln - W / S);
    for (int64_t c = threadIdx.x; c < a.C; c += kLpThreads) {
        const int64_t t = a.targets[n * a.C + c];
        float r;
        if (t < 0) r = 0.f;
        else if (t >= a.V || is_bad) r = NAN;
        else if (none || gone(t)) r = -INFINITY;
        else r = lp_float(x[t]) * a.scale - m - ln;
        a.lp[n * a.C + c] = r;
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < a.top; ++k) {
        uint64_t next = 0;
        if (!is_bad)
            for (int i = threadIdx.x; i < a.V; i += kLpThreads) {
                const float v = lp_float(x[i]);
                if (gone(i) || !(v > -INFINITY)) continue;
                const uint64_t key = lp_key(v, i);
                if (key < last) next = most(next, key);
            }
        next = lp_block_reduce(next, most, red_k);
        if (threadIdx.x == 0) {
            a.top_ids[n * a.top + k] = next ? (int64_t)(uint32_t)~(uint32_t)next : -1;
            a.top_lp[n * a.top + k] = is_bad ? NAN : (next ? lp_key_value(next) * a.scale - m - ln : -INFINITY);
        }
        last = next;
    }
}

cudaError_t token_logprobs(const LogprobsArgs &a, cudaStream_t st) {
    const dim3 grid((unsigned)a.N), block(kLpThreads);
    switch (a.dtype) {
        case 0: return launch_pdl(token_logprobs_kernel<int8_t>, grid, block, 0, st, a);
        case 1: return launch_pdl(token_logprobs_kernel<__half>, grid, block, 0, st, a);
        case 2: return launch_pdl(token_logprobs_kernel<__nv_bfloat16>, grid, block, 0, st, a);
        default: return launch_pdl(token_logprobs_kernel<float>, grid, block, 0, st, a);
    }
}

}  // namespace iw
