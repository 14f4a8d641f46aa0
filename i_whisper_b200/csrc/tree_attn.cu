// tree_attn.cu -- integer attention of ragged drafted trees over a paged INT8
// cache (iw_tree_attention). With x = sat16(rrs(q.k * m, s)) for the keys that
// a row sees and M their maximum,
//   p = shift_exp(x - M - 1),  o = clamp(rrs(rrs(rrs(sum p v * i, f) * i, f) * am, as)),
//   i = fisr(sum p)  with f = rsqrt_offset,
// the steps of the dense attention (kernels.cu). All sums are integers, so how
// the keys are split does not change a bit of the result.
#include "iw_common.cuh"
#include "paged.cuh"

namespace iw {

// One warp per (new token, query head): keys across lanes for the scores,
// channels across lanes for P.V; the keys are read twice.
template <int D>
__global__ void __launch_bounds__(128) tree_attn_kernel(TreeAttnArgs a) {
    pdl_wait();
    pdl_launch();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= a.N * a.H) return;
    const int64_t n = row / a.H;
    const int h = (int)(row - n * a.H), kvh = h / (a.H / a.Hkv);
    int8_t *out = a.y + n * a.ldy + (int64_t)h * D;
    if (n >= a.starts[a.B]) {
        for (int d = lane; d < D; d += 32) out[d] = 0;
        return;
    }
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.starts[mid] <= n) lo = mid;
        else hi = mid - 1;
    }
    const int b = lo;
    const int t = (int)(n - a.starts[b]);
    const int fresh = a.starts[b + 1] - a.starts[b];
    const int ctx = max(a.ctx[b], 0);
    const int64_t cap = (int64_t)a.width << a.page_log2;
    const int L = (int)min((int64_t)ctx + fresh, cap);
    const int32_t *tab = a.table + (int64_t)b * a.table_ld;
    int4 q[D / 16];
#pragma unroll
    for (int c = 0; c < D / 16; ++c) q[c] = *reinterpret_cast<const int4 *>(a.q + n * a.ldq + h * a.q_hs + 16 * c);
    auto place = [&](int j) -> int64_t {  // byte offset of key j's row, -1 when it has no page
        const int32_t page = tab[j >> a.page_log2];
        if (page < 0 || page >= a.n_pages) return -1;
        return page * a.page_stride + kvh * a.head_stride + (j & ((1 << a.page_log2) - 1)) * a.row_stride;
    };
    auto score = [&](int j, int32_t &x) -> bool {
        if (j >= L) return false;
        const int u = j - ctx;
        if (u >= 0) {
            if (a.words) {
                if ((u >> 5) >= a.words || !((a.mask[n * a.words + (u >> 5)] >> (u & 31)) & 1)) return false;
            } else if (u > t) {
                return false;
            }
        }
        const int64_t at = place(j);
        if (at < 0) return false;
        int32_t acc = 0;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            const int4 k = *reinterpret_cast<const int4 *>(a.k + at + 16 * c);
            acc = __dp4a(k.x, q[c].x, acc);
            acc = __dp4a(k.y, q[c].y, acc);
            acc = __dp4a(k.z, q[c].z, acc);
            acc = __dp4a(k.w, q[c].w, acc);
        }
        x = clampi(rrs(wmul(acc, a.qk_mult), a.qk_shift), -32768, 32767);
        return true;
    };
    int32_t m = -32768;
    for (int j = lane; j < L; j += 32) {
        int32_t x;
        if (score(j, x)) m = max(m, x);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    const int32_t xm = (int16_t)(m + 1);
    int32_t sum = 0;
    uint32_t acc[D / 32];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = 0;
    for (int j0 = 0; j0 < L; j0 += 32) {
        int32_t x, p = 0;
        if (score(j0 + lane, x)) p = shift_exp_one(x, xm, a.frac_bits);
        sum += p;
        uint32_t some = __ballot_sync(0xffffffffu, p != 0);
        while (some) {
            const int s = __ffs(some) - 1;
            some &= some - 1;
            const int32_t ps = __shfl_sync(0xffffffffu, p, s);
            const int8_t *vr = a.v + place(j0 + s) + lane * (D / 32);
#pragma unroll
            for (int e = 0; e < D / 32; ++e) acc[e] += (uint32_t)(ps * (int32_t)vr[e]);
        }
    }
    sum = __reduce_add_sync(0xffffffffu, sum);
    const int32_t inv = fisr(sum, a.rsqrt_offset);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) {
        int32_t v = rrs(wmul((int32_t)acc[e], inv), a.rsqrt_offset);
        v = rrs(wmul(v, inv), a.rsqrt_offset);
        v = rrs(wmul(v, a.av_mult), a.av_shift);
        out[lane * (D / 32) + e] = (int8_t)clampi(v, -127, 127);
    }
}

cudaError_t tree_attention(const TreeAttnArgs &a, cudaStream_t st) {
    const int64_t blocks = (a.N * a.H + 3) / 4;
    if (a.D == 64) return launch_pdl(tree_attn_kernel<64>, dim3((unsigned)blocks), dim3(128), 0, st, a);
    return launch_pdl(tree_attn_kernel<128>, dim3((unsigned)blocks), dim3(128), 0, st, a);
}

}  // namespace iw
