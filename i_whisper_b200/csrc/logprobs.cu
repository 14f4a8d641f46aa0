// logprobs.cu -- log probabilities of given tokens, entropy and the most
// likely tokens of each row of logits (iw_token_logprobs). With l = scale * x
// over the tokens that are not suppressed, m = max l and S = sum exp(l - m),
//   lp(t) = l_t - m - ln S,   H = ln S - sum (l - m) exp(l - m) / S.
//
// One block per row reads it once, 16 bytes per thread and load.
//   Floating types: each thread keeps a running maximum and the sums relative to
//   it, rescaled when the maximum moves; in units of log 2, so that the
//   exponential is one instruction. Bound by issue at 16 bits, a dozen instructions per
//   element with suppressed ids: 1031 rows of 100003 bf16 logits, 3 given tokens, 20
//   alternatives, 70 us, 3.0 TB/s, and 59 us without suppressed ids.
//   int8: there are 256 logits, so the row's histogram says it all: each lane
//   counts into a column of its own (bank = lane, no conflicts), and the sums
//   are taken over 256 exact counts. Bound by the rate of shared-memory
//   additions: 4096 rows of 51865 logits, 5 alternatives, 64 us, 3.3 TB/s (54 without
//   alternatives, 75 with suppressed ids); an exponential per element measured 16 us
//   more.
// The most likely tokens: each thread knows its own maximum, so at least
// `top` elements reach the top-th largest of these; the few elements that do
// are fetched again (a warp per thread that has some) and ranked among
// themselves. Rows in which too many do (ties) take a pass per alternative.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "iw_common.cuh"
#include "paged.cuh"

namespace iw {
namespace lp {

constexpr int kCandidates = 512;
// Threads per block where the rows fill the GPU: int8 rows want few, since each
// block zeroes and sums its histogram once (512 measured a quarter slower), the
// others 512 (256 measured a fifth slower). Fewer rows than SMs leave
// room for 1024 each.
template <typename T>
constexpr int threads_of() { return sizeof(T) == 1 ? 256 : 512; }
constexpr int kThreadsFewRows = 1024;

IW_DEV float to_float(int8_t v) { return (float)v; }
IW_DEV float to_float(float v) { return v; }
IW_DEV float to_float(__half v) { return __half2float(v); }
IW_DEV float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Two 16-bit floats of a word.
IW_DEV void widen(__nv_bfloat16, uint32_t w, float &lo, float &hi) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
}
IW_DEV void widen(__half, uint32_t w, float &lo, float &hi) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    lo = v.x, hi = v.y;
}

// The elements of a 16-byte vector.
template <typename T>
IW_DEV void unpack(const int4 &w, float (&f)[16 / sizeof(T)]) {
    const uint32_t q[4] = {(uint32_t)w.x, (uint32_t)w.y, (uint32_t)w.z, (uint32_t)w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 4) f[e] = __uint_as_float(q[e]);
        else if constexpr (sizeof(T) == 2) widen(T(), q[e], f[2 * e], f[2 * e + 1]);
        else
#pragma unroll
            for (int b = 0; b < 4; ++b) f[4 * e + b] = (float)(int8_t)(q[e] >> (8 * b));
    }
}

IW_DEV float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A float's bits made to order as an unsigned number; zeros are equal.
IW_DEV uint32_t order(float v) {
    const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
IW_DEV float unorder(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }
// Rank of (value, id): larger is better, the lower id first.
IW_DEV uint64_t key_of(float v, uint32_t id) { return ((uint64_t)order(v) << 32) | (uint32_t)~id; }

template <int kThreads, typename F, typename T>
IW_DEV T block_reduce(T v, F f, T *red) {
    constexpr int kWarps = kThreads / 32;
    __syncthreads();
#pragma unroll
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[threadIdx.x & (kWarps - 1)];
#pragma unroll
    for (int o = kWarps / 2; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// A row cut into 16-byte vectors: `head` elements before the first aligned one,
// `vecs` vectors, `tail` elements. Vector v belongs to thread v % (threads),
// head and tail elements, fewer than 16 each, to the first `head + tail` threads.
template <typename T>
struct Row {
    static constexpr int kPer = 16 / sizeof(T);
    const T *x;
    int V, head, vecs, tail;
    IW_DEV Row(const T *x_, int V_) : x(x_), V(V_) {
        const int misaligned = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
        head = min(V, misaligned ? kPer - misaligned : 0);
        vecs = (V - head) / kPer;
        tail = V - head - vecs * kPer;
    }
    IW_DEV int first(int v) const { return head + v * kPer; }
    IW_DEV int4 load(int v) const { return *reinterpret_cast<const int4 *>(x + first(v)); }
    // index of the thread's element outside the vectors, -1 for none
    IW_DEV int edge(int t) const { return t < head ? t : (t < head + tail ? t + vecs * kPer : -1); }
};

// The thread's vectors, U loads in flight at a time.
template <int kThreads, int U, typename T, typename F>
IW_DEV void for_vectors(const Row<T> &row, int tid, F f) {
    int v = tid;
#pragma unroll 1
    for (; v + (U - 1) * kThreads < row.vecs; v += U * kThreads) {
        int4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = row.load(v + u * kThreads);
#pragma unroll
        for (int u = 0; u < U; ++u) f(v + u * kThreads, w[u]);
    }
#pragma unroll 1
    for (; v < row.vecs; v += kThreads) f(v, row.load(v));
}

// kPer suppression bits from element i on.
template <int N>
IW_DEV uint32_t bits_at(const uint32_t *bits, int i, int V) {
    const int w = i >> 5, last = (V - 1) >> 5;
    return __funnelshift_r(__ldg(bits + w), __ldg(bits + min(w + 1, last)), i & 31) & ((1u << N) - 1);
}

template <int kThreads>
struct Shared {
    float red[kThreads / 32];
    uint64_t red64[kThreads / 32];
    uint64_t cand[kCandidates];
    uint16_t owners[kThreads];
    int n_cand, n_owners, n_gone;
    uint32_t bins[256], at_least, threshold;  // int8
    float m, S, W;
};

// Larger of two, NaN when either is.
IW_DEV float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

template <typename T, bool SUP, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == 1024 ? 1 : (sizeof(T) == 1 ? 5 : 3)) token_logprobs_kernel(LogprobsArgs a) {
    // int8: five blocks' histograms fill an SM's shared memory
    static_assert(kThreads >= 32, "a thread for every element outside the vectors");
    constexpr bool kBytes = sizeof(T) == 1;
    constexpr int P = Row<T>::kPer, kWarps = kThreads / 32;
    pdl_wait();
    pdl_launch();
    extern __shared__ uint32_t hist[];  // int8: [256][32]
    __shared__ Shared<kThreads> s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t n = blockIdx.x;
    const Row<T> row(reinterpret_cast<const T *>(a.x) + n * a.ld, a.V);
    auto gone = [&](int i) { return SUP && ((__ldg(a.suppress + (i >> 5)) >> (i & 31)) & 1u); };
    auto most = [](float p, float q) { return fmaxf(p, q); };
    auto add = [](float p, float q) { return p + q; };
    const float c = a.scale * 1.4426950408889634f;  // scale / ln 2
    if (tid == 0) s.n_cand = s.n_owners = s.n_gone = 0;

    float mine = -INFINITY;   // the thread's largest logit
    float m, S, W;            // of the row: maximum (unscaled), sum of 2^t, sum of t 2^t with t = c (x - m)
    uint32_t at_least = 0;    // elements that reach the threshold (int8)
    uint32_t threshold = 0;   // order() of the smallest value that may be among the best
    if constexpr (kBytes) {
        for (int i = tid; i < 256 * 32 / 4; i += kThreads) reinterpret_cast<int4 *>(hist)[i] = make_int4(0, 0, 0, 0);
        __syncthreads();
        const uint32_t column = (uint32_t)__cvta_generic_to_shared(hist) + lane * 4;
        uint32_t even = 0, odd = 0;  // largest x + 128 of the bytes 0, 2 and 1, 3, 16 bits each
        auto count = [&](uint32_t u) { asm volatile("red.shared.add.u32 [%0], 1;" ::"r"(column + u * 128)); };
        int n_gone = 0;
        auto words = [&](uint32_t w, uint32_t x) {
#pragma unroll
            for (int e = 0; e < 4; ++e) count(__byte_perm(w, 0, 0x4440 + e));
#pragma unroll
            for (int e = 0; e < 4; ++e) count(__byte_perm(x, 0, 0x4440 + e));
            even = __vimax3_u16x2(even, w & 0x00ff00ffu, x & 0x00ff00ffu);
            odd = __vimax3_u16x2(odd, __byte_perm(w, 0, 0x4341), __byte_perm(x, 0, 0x4341));
        };
        auto vector = [&](int v, const int4 &q) {
            uint32_t w[4] = {(uint32_t)q.x ^ 0x80808080u, (uint32_t)q.y ^ 0x80808080u, (uint32_t)q.z ^ 0x80808080u,
                             (uint32_t)q.w ^ 0x80808080u};
            if (SUP) {
                // suppressed bytes count as the smallest value, and are taken off that count below
                const uint32_t sup = bits_at<16>(a.suppress, row.first(v), a.V);
                n_gone += __popc(sup);
#pragma unroll
                for (int e = 0; e < 4; ++e)  // four bits to four bytes
                    w[e] &= ~((((sup >> (4 * e) & 15) * 0x00204081u) & 0x01010101u) * 255u);
            }
            words(w[0], w[1]), words(w[2], w[3]);
        };
        for_vectors<kThreads, 4>(row, tid, vector);
        const int e = row.edge(tid);
        const bool extra = e >= 0 && !gone(e);
        if (extra) {
            const uint32_t u = (uint32_t)((int)row.x[e] + 128);
            count(u);
            even = __vimax3_u16x2(even, u, 0);
        }
        mine = (float)(int)max(max(even & 0xffffu, even >> 16), max(odd & 0xffffu, odd >> 16)) - 128.f;
        if (SUP) {
            n_gone = __reduce_add_sync(0xffffffffu, n_gone);
            if (lane == 0) atomicAdd(&s.n_gone, n_gone);
        }
        __syncthreads();
        {  // a thread per value; its 32 counters in an order free of bank conflicts
            uint32_t cnt = 0;
            if (tid < 256) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint4 q = reinterpret_cast<const uint4 *>(hist)[tid * 8 + ((j + lane) & 7)];
                    cnt += q.x + q.y + q.z + q.w;
                }
                if (SUP && tid == 0) cnt -= s.n_gone;
                s.bins[255 - tid] = cnt;  // from the largest value down
            }
        }
        __syncthreads();
        if (warp == 0) {  // lane: the values 127 - 8 * lane .. 120 - 8 * lane
            uint32_t cnt[8], sum = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += cnt[j] = s.bins[8 * lane + j];
            uint32_t upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += t;
            }
            int top = -1000;
#pragma unroll
            for (int j = 7; j >= 0; --j)
                if (cnt[j]) top = 127 - 8 * lane - j;
            top = __reduce_max_sync(0xffffffffu, top);
            float Sm = 0.f, Wm = 0.f;
            // the value at which the count first reaches `top` (-128 if it never does)
            uint32_t before = upto - sum, reached = 0;
            int low = -128;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int value = 127 - 8 * lane - j;
                if (cnt[j]) {
                    const float t = c * (float)(value - top), ex = (float)cnt[j] * exp2f(t);
                    Sm += ex;
                    Wm = fmaf(ex, t, Wm);
                }
                if (before < (uint32_t)a.top && before + cnt[j] >= (uint32_t)a.top) low = value, reached = before + cnt[j];
                before += cnt[j];
            }
            const uint32_t total = __shfl_sync(0xffffffffu, upto, 31);
            low = __reduce_max_sync(0xffffffffu, low);
            reached = __reduce_max_sync(0xffffffffu, reached);
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                Sm += __shfl_xor_sync(0xffffffffu, Sm, o);
                Wm += __shfl_xor_sync(0xffffffffu, Wm, o);
            }
            if (lane == 0) {
                s.m = total ? (float)top : -INFINITY;
                s.S = Sm, s.W = Wm;
                s.at_least = reached ? reached : total;
                s.threshold = order((float)low);
            }
        }
        __syncthreads();
        m = s.m, S = s.S, W = s.W;
        at_least = s.at_least, threshold = s.threshold;
    } else {
        float Sm = 0.f, Wm = 0.f, ref = 0.f;  // ref: mine, or 0 before there is one
        auto take = [&](const float (&v)[P]) {
            float top = v[0];
#pragma unroll
            for (int e = 1; e < P; ++e) top = fmaxf(top, v[e]);
            if (top > mine) {
                const float d = mine > -INFINITY ? fmaxf(c * (mine - top), -200.f) : 0.f, f = exp2_approx(d);
                Wm = (Wm + d * Sm) * f;
                Sm *= f;
                mine = ref = top;
            }
#pragma unroll
            for (int e = 0; e < P; ++e) {
                // far below the maximum, or -inf: 2^-200, which is 0; a NaN passes as NaN
                const float t = max_nan(c * (v[e] - ref), -200.f), ex = exp2_approx(t);
                Sm += ex;
                Wm = fmaf(ex, t, Wm);
            }
        };
        auto vector = [&](int v, const int4 &w) {
            float f[P];
            unpack<T>(w, f);
            if (SUP) {
                const uint32_t sup = bits_at<P>(a.suppress, row.first(v), a.V);
                if (sup) {
#pragma unroll
                    for (int e = 0; e < P; ++e)
                        if ((sup >> e) & 1) f[e] = -INFINITY;
                }
            }
            take(f);
        };
        for_vectors<kThreads, 2>(row, tid, vector);
        const int e = row.edge(tid);
        if (e >= 0 && !gone(e)) {
            float f[P];
            f[0] = to_float(row.x[e]);
#pragma unroll
            for (int k = 1; k < P; ++k) f[k] = -INFINITY;
            take(f);
        }
        m = block_reduce<kThreads>(mine, most, s.red);
        const float d = mine > -INFINITY ? fmaxf(c * (mine - m), -200.f) : 0.f, f = exp2_approx(d);
        S = block_reduce<kThreads>(Sm * f, add, s.red);
        W = block_reduce<kThreads>((Wm + d * Sm) * f, add, s.red);
    }
    // a NaN makes S NaN, and so does +inf, from which nothing finite can be taken
    const bool bad = !(S >= 0.f) || m == INFINITY;
    const bool none = !bad && m == -INFINITY;
    const float log2S = log2f(S);
    constexpr float kLn2 = 0.6931471805599453f;
    auto log_prob = [&](float x) { return a.scale * (x - m) - kLn2 * log2S; };
    if (tid == 0) a.entropy[n] = bad ? NAN : (none ? 0.f : kLn2 * (log2S - W / S));
    for (int64_t k = tid; k < a.C; k += kThreads) {
        const int64_t t = a.targets[n * a.C + k];
        float r;
        if (t < 0) r = 0.f;
        else if (t >= a.V || bad) r = NAN;
        else if (none || gone((int)t) || !(to_float(row.x[t]) > -INFINITY)) r = -INFINITY;
        else r = log_prob(to_float(row.x[t]));
        a.lp[n * a.C + k] = r;
    }
    if (a.top == 0) return;
    int64_t *ids = a.top_ids + n * a.top;
    float *lps = a.top_lp + n * a.top;
    if (bad || none) {
        for (int k = tid; k < a.top; k += kThreads) ids[k] = -1, lps[k] = bad ? NAN : -INFINITY;
        return;
    }
    bool slow = false;
    if constexpr (kBytes) {
        slow = at_least > kCandidates;
    } else {
        // the largest 16-bit prefix that the maxima of `top` threads reach
        const uint32_t o = mine > -INFINITY ? order(mine) >> 16 : 0;
        uint32_t p = 0;
#pragma unroll 1
        for (int b = 15; b >= 0; --b)
            if (__syncthreads_count(o >= (p | (1u << b))) >= a.top) p |= 1u << b;
        threshold = p << 16;
    }
    if (!slow) {
        if (mine > -INFINITY && order(mine) >= threshold) s.owners[atomicAdd(&s.n_owners, 1)] = (uint16_t)tid;
        __syncthreads();
        auto offer = [&](int i, float v) {
            if (!(v > -INFINITY) || order(v) < threshold || gone(i)) return;
            const int at = atomicAdd(&s.n_cand, 1);
            if (at < kCandidates) s.cand[at] = key_of(v, i);
        };
        // a warp per such thread: its lanes take the thread's vectors
        const int owners = s.n_owners;
        for (int k = warp; k < owners; k += kWarps) {
            const int t = s.owners[k];
            for (int v = t + lane * kThreads; v < row.vecs; v += 32 * kThreads) {
                float f[P];
                unpack<T>(row.load(v), f);
#pragma unroll
                for (int e = 0; e < P; ++e) offer(row.first(v) + e, f[e]);
            }
            const int e = row.edge(t);
            if (lane == 0 && e >= 0) offer(e, to_float(row.x[e]));
        }
        __syncthreads();
        const int found = s.n_cand;
        slow = found > kCandidates;
        if (!slow) {
            for (int k = tid; k < max(found, a.top); k += kThreads) {
                if (k >= found) {
                    if (k < a.top) ids[k] = -1, lps[k] = -INFINITY;
                    continue;
                }
                const uint64_t key = s.cand[k];
                int rank = 0;
                for (int j = 0; j < found; ++j) rank += s.cand[j] > key;
                if (rank < a.top) {
                    ids[rank] = (int64_t)(uint32_t)~(uint32_t)key;
                    lps[rank] = log_prob(unorder((uint32_t)(key >> 32)));
                }
            }
        }
    }
    if (slow) {
        uint64_t last = ~0ull;
        for (int k = 0; k < a.top; ++k) {
            uint64_t next = 0;
            for (int i = tid; i < a.V; i += kThreads) {
                const float v = to_float(row.x[i]);
                if (gone(i) || !(v > -INFINITY)) continue;
                const uint64_t key = key_of(v, i);
                if (key < last && key > next) next = key;
            }
            next = block_reduce<kThreads>(next, [](uint64_t p, uint64_t q) { return p > q ? p : q; }, s.red64);
            if (tid == 0) {
                ids[k] = next ? (int64_t)(uint32_t)~(uint32_t)next : -1;
                lps[k] = next ? log_prob(unorder((uint32_t)(next >> 32))) : -INFINITY;
            }
            last = next;
        }
    }
}

template <typename T, int kThreads>
static cudaError_t launch_threads(const LogprobsArgs &a, cudaStream_t st) {
    const size_t smem = sizeof(T) == 1 ? 256 * 32 * 4 : 0;
    const dim3 grid((unsigned)a.N), block(kThreads);
    return a.suppress ? launch_pdl(token_logprobs_kernel<T, true, kThreads>, grid, block, smem, st, a)
                      : launch_pdl(token_logprobs_kernel<T, false, kThreads>, grid, block, smem, st, a);
}
template <typename T>
static cudaError_t launch(const LogprobsArgs &a, cudaStream_t st) {
    return a.N <= num_sms() ? launch_threads<T, kThreadsFewRows>(a, st) : launch_threads<T, threads_of<T>()>(a, st);
}

}  // namespace lp

cudaError_t token_logprobs(const LogprobsArgs &a, cudaStream_t st) {
    switch (a.dtype) {
        case 0: return lp::launch<int8_t>(a, st);
        case 1: return lp::launch<__half>(a, st);
        case 2: return lp::launch<__nv_bfloat16>(a, st);
        default: return lp::launch<float>(a, st);
    }
}

}  // namespace iw
