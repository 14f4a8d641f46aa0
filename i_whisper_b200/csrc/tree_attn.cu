// tree_attn.cu -- integer attention of ragged drafted trees over a paged INT8
// cache (iw_tree_attention). With x = sat16(rrs(q.k * m, s)) for the keys that
// a row sees and M their maximum,
//   p = shift_exp(x - M - 1),  o = clamp(rrs(rrs(rrs(sum p v * i, f) * i, f) * am, as)),
//   i = fisr(sum p)  with f = rsqrt_offset,
// the steps of the dense attention (kernels.cu). All sums are integers, so how
// the keys are split does not change a bit of the result.
#include <cooperative_groups.h>

#include "iw_common.cuh"
#include "paged.cuh"

namespace iw {
namespace tree {

constexpr int kSlab = 32;  // keys per step of a warp

// c += a (16 rows x 32, signed or unsigned bytes) * b (32 x 8 signed bytes).
// Lane (g = lane/4, t = lane%4) holds a0/a1: rows g/g+8, k 4t..4t+3, a2/a3:
// the same rows, k 16+4t..; b0/b1: column g, k 4t.. / 16+4t..; c0,c1/c2,c3:
// rows g/g+8, columns 2t, 2t+1.
IW_DEV void mma_s8(int32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
IW_DEV void mma_u8s8(int32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two 16 x 16 byte tiles, transposed: lanes 0-15 point at the rows of the
// first, 16-31 at those of the second; r0/r1: rows 4t..4t+3 of columns g / 8+g
// of the first tile, r2/r3 of the second.
IW_DEV void ldsm_trans_b8(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(p))
                 : "memory");
}

// What one request asks for, the same in every block that serves it.
struct Request {
    int first, fresh;  // rows of its new tokens
    int ctx, keys;     // cached tokens; keys in all, cut to the block table
    const int32_t *table;
};
IW_DEV Request request(const TreeAttnArgs &a, int b) {
    Request r;
    const int64_t s0 = a.starts[b], s1 = a.starts[b + 1];
    r.first = (int)s0;
    r.fresh = (s0 < 0 || s1 <= s0 || s0 >= a.N) ? 0 : (int)(min(s1, a.N) - s0);
    r.ctx = max(a.ctx[b], 0);
    r.keys = (int)min((int64_t)r.ctx + r.fresh, (int64_t)a.width << a.page_log2);
    r.table = a.table + (int64_t)b * a.table_ld;
    return r;
}

// Byte offset of key j's row of one head in the caches, -1 when it has no page.
IW_DEV int64_t key_row(const TreeAttnArgs &a, const Request &r, int64_t head_at, int j) {
    if (j >= r.keys) return -1;
    const int32_t page = r.table[j >> a.page_log2];
    if ((uint32_t)page >= (uint32_t)a.n_pages) return -1;
    return page * a.page_stride + head_at + (j & ((1 << a.page_log2) - 1)) * a.row_stride;
}

// Whether new token t of the request sees key j, which has a page.
IW_DEV bool sees(const TreeAttnArgs &a, const Request &r, int t, int j) {
    const int u = j - r.ctx;
    if (u < 0) return true;
    if (a.words == 0) return u <= t;
    return (u >> 5) < a.words && ((a.mask[(int64_t)(r.first + t) * a.words + (u >> 5)] >> (u & 31)) & 1);
}

IW_DEV int32_t finish(const TreeAttnArgs &a, int32_t acc, int32_t inv) {
    int32_t v = rrs(wmul(acc, inv), a.rsqrt_offset);
    v = rrs(wmul(v, inv), a.rsqrt_offset);
    v = rrs(wmul(v, a.av_mult), a.av_shift);
    return clampi(v, -127, 127);
}

// Rows from starts[B] on are padding: the blocks of the last request zero
// them, each its own heads.
IW_DEV void zero_padding(const TreeAttnArgs &a, int kvh, int rank, int ranks) {
    const int64_t first = max(a.starts[a.B], 0);
    const int G = a.H / a.Hkv, per = G * a.D / 16;
    for (int64_t i = (int64_t)rank * blockDim.x + threadIdx.x; i < (a.N - first) * per; i += (int64_t)ranks * blockDim.x)
        *reinterpret_cast<int4 *>(a.y + (first + i / per) * a.ldy + (int64_t)kvh * G * a.D + (i % per) * 16) =
            make_int4(0, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// Few rows per key head (single tokens, small trees): bound by reading K and V
// once from HBM. A cluster of blocks serves one (request, key head) and
// splits its keys; each warp streams slabs of 32 keys through a ring of its
// own (cp.async, no block barrier), K first: 16 rows by 32 scores by
// mma.sync, requantised scores kept in shared memory as 16 bits, so that K is
// not read again once the maximum over all blocks is known (exchanged
// through distributed shared memory); then V: probabilities, one thread per
// (row, key), and P.V by mma.sync with V transposed by ldmatrix. mma.sync and
// not tcgen05: with at most 16 rows the 128-row tile would be padding, and
// the tensor pipe is far from the limit at HBM rate.
// ---------------------------------------------------------------------------
constexpr int kFewWarps = 4;
constexpr int kScoreLd = 80;  // bytes per row of a slab's scores: 32 x 16 bits, padded against bank conflicts

template <int D>
struct Few {
    static constexpr int kStages = D == 64 ? 4 : 3;
    static constexpr int kRing = kStages * kSlab * D;
    static size_t smem(int score_cap) { return (size_t)kFewWarps * (kRing + score_cap) + 16 * D * 4 + 32 * 4; }
};

// 16-byte pieces of a slab's rows are swizzled so that the fragment loads are
// free of bank conflicts: K (one int4 per lane, two rows of 64 bytes a
// quarter warp) needs it at 128-byte rows, V (16 rows of one piece) at both.
template <int D>
IW_DEV int k_piece(int row, int c) { return D == 64 ? c : c ^ ((row & 1) << 2); }
template <int D>
IW_DEV int v_piece(int row, int c) { return D == 64 ? c ^ ((row >> 1) & 3) : c ^ (row & 7); }

template <int D>
__global__ void __launch_bounds__(32 * kFewWarps) few_rows_kernel(TreeAttnArgs a, int score_cap) {
    namespace cg = cooperative_groups;
    pdl_wait();
    pdl_launch();
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    constexpr int S = Few<D>::kStages;
    uint8_t *ring = smem + warp * Few<D>::kRing;
    uint8_t *score = smem + kFewWarps * Few<D>::kRing + warp * score_cap;
    int32_t *s_o = reinterpret_cast<int32_t *>(smem + kFewWarps * (Few<D>::kRing + score_cap));  // [16][D]
    int32_t *s_max = s_o + 16 * D, *s_sum = s_max + 16;
    const int rank = blockIdx.x, ranks = gridDim.x, kvh = blockIdx.y, b = blockIdx.z;
    const int G = a.H / a.Hkv;
    if (b == a.B - 1) zero_padding(a, kvh, rank, ranks);
    const Request r = request(a, b);
    const int rows = r.fresh * G;
    if (rows == 0) return;
    const int64_t head_at = (int64_t)kvh * a.head_stride;
    const int slabs = (r.keys + kSlab - 1) / kSlab;
    const int first = (int)((int64_t)slabs * rank / ranks), last = (int)((int64_t)slabs * (rank + 1) / ranks);
    const int mine = max(0, (last - first - warp + kFewWarps - 1) / kFewWarps);
    auto slab_at = [&](int i) { return (first + warp + i * kFewWarps) * kSlab; };
    const RrsK rk = rrs_k(a.qk_shift);

    for (int row0 = 0; row0 < rows; row0 += 16) {
        const int nr = min(16, rows - row0);
        const bool keep = mine * nr * kScoreLd <= score_cap;
        // the stream of slabs: K0 .. Kn-1, then V0 .. Vn-1, or K0 V0 K1 V1 ... when
        // the scores could not be kept
        const int items = mine * (keep ? 2 : 3);
        auto issue = [&](int it) {
            if (it < items) {
                const bool v = keep ? it >= mine : (it >= mine && ((it - mine) & 1));
                const int i = it < mine ? it : (keep ? it - mine : (it - mine) >> 1);
                const int j0 = slab_at(i);
                const int8_t *src = v ? a.v : a.k;
                uint8_t *dst = ring + (it % S) * (kSlab * D);
#pragma unroll
                for (int e = 0; e < D / 16; ++e) {
                    const int row = (e * 32 + lane) / (D / 16), c = lane % (D / 16);
                    const int64_t at = key_row(a, r, head_at, j0 + row);
                    uint8_t *to = dst + row * D + (v ? v_piece<D>(row, c) : k_piece<D>(row, c)) * 16;
                    if (at >= 0) cp_async16(to, src + at + 16 * c);
                    else *reinterpret_cast<int4 *>(to) = make_int4(0, 0, 0, 0);
                }
            }
            cp_async_commit();
        };
        for (int i = 0; i < S; ++i) issue(i);

        // queries: lane's 16 bytes of rows g and g+8 in each 64-byte half, so that
        // bytes 8s.. and 8s+4.. of the piece are a0 and a2 of step s
        int4 q0[D / 64], q1[D / 64];
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
            q0[c] = q1[c] = make_int4(0, 0, 0, 0);
            const int ra = row0 + g, rb = ra + 8;
            if (ra < rows)
                q0[c] = *reinterpret_cast<const int4 *>(a.q + (int64_t)(r.first + ra / G) * a.ldq +
                                                        (int64_t)(kvh * G + ra % G) * a.q_hs + 64 * c + 16 * t);
            if (rb < rows)
                q1[c] = *reinterpret_cast<const int4 *>(a.q + (int64_t)(r.first + rb / G) * a.ldq +
                                                        (int64_t)(kvh * G + rb % G) * a.q_hs + 64 * c + 16 * t);
        }
        for (int i = tid; i < 16 * D + 32; i += 32 * kFewWarps) s_o[i] = i >= 16 * D && i < 16 * D + 16 ? -32768 : 0;
        __syncthreads();

        int32_t m0 = -32768, m1 = -32768, mr = -32768;  // rows g, g + 8 (own columns); row = lane (masked slabs)
        // whether every row sees every key of the slab, and which keys have a page
        auto plain_slab = [&](int j0, uint32_t &there) {
            there = __ballot_sync(0xffffffffu, key_row(a, r, head_at, j0 + lane) >= 0);
            return there == 0xffffffffu && j0 + kSlab <= r.ctx;
        };
        // scores of a K slab in the ring -> score slot, and the running maximum
        auto scores = [&](const uint8_t *ks, int j0, uint8_t *to, bool want_max, bool store) {
            uint32_t there;
            const bool plain = plain_slab(j0, there);
#pragma unroll
            for (int n8 = 0; n8 < 4; ++n8) {
                int32_t c[4] = {0, 0, 0, 0};
#pragma unroll
                for (int h = 0; h < D / 64; ++h) {
                    const int row = 8 * n8 + g;
                    const int4 k = *reinterpret_cast<const int4 *>(ks + row * D + k_piece<D>(row, 4 * h + t) * 16);
                    mma_s8(c, q0[h].x, q1[h].x, q0[h].y, q1[h].y, k.x, k.y);
                    mma_s8(c, q0[h].z, q1[h].z, q0[h].w, q1[h].w, k.z, k.w);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) c[e] = clampi(rrs_apply(wmul(c[e], a.qk_mult), rk), -32768, 32767);
                if (plain) {
                    m0 = max(m0, max(c[0], c[1]));
                    m1 = max(m1, max(c[2], c[3]));
                }
                if (store || !plain) {
                    uint8_t *w = to + 16 * n8 + 4 * t;
                    if (g < nr) *reinterpret_cast<uint32_t *>(w + g * kScoreLd) = __byte_perm(c[0], c[1], 0x5410);
                    if (g + 8 < nr) *reinterpret_cast<uint32_t *>(w + (g + 8) * kScoreLd) = __byte_perm(c[2], c[3], 0x5410);
                }
            }
            __syncwarp();
            if (want_max && !plain) {
                for (int i = 0; i < nr; ++i) {
                    const bool on = ((there >> lane) & 1) && sees(a, r, (row0 + i) / G, j0 + lane);
                    const int32_t x = *reinterpret_cast<const int16_t *>(to + i * kScoreLd + 2 * lane);
                    const int32_t m = __reduce_max_sync(0xffffffffu, on ? x : -32768);
                    if (lane == i) mr = max(mr, m);
                }
                __syncwarp();
            }
        };
        int it = 0;
        for (int i = 0; i < mine; ++i, ++it) {
            cp_async_wait<S - 1>();
            __syncwarp();
            scores(ring + (it % S) * (kSlab * D), slab_at(i), score + (keep ? i * nr * kScoreLd : 0), true, keep);
            issue(it + S);
        }
        // row maxima: over the lanes, the warps, the cluster
        m0 = max(m0, __shfl_xor_sync(0xffffffffu, m0, 1));
        m1 = max(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
        m0 = max(m0, __shfl_xor_sync(0xffffffffu, m0, 2));
        m1 = max(m1, __shfl_xor_sync(0xffffffffu, m1, 2));
        if (t == 0) atomicMax(&s_max[g], m0), atomicMax(&s_max[g + 8], m1);
        if (lane < nr) atomicMax(&s_max[lane], mr);
        int32_t xm = -32768;  // row = lane
        if (ranks == 1) {
            __syncthreads();
            if (lane < 16) xm = s_max[lane];
        } else {
            cg::cluster_group cl = cg::this_cluster();
            cl.sync();
            if (lane < 16)
                for (int k = 0; k < ranks; ++k) xm = max(xm, cl.map_shared_rank(s_max, k)[lane]);
        }
        xm = (int16_t)(xm + 1);

        int32_t o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0;
        int32_t sum0 = 0, sum1 = 0;
        for (int i = 0; i < mine; ++i) {
            const int j0 = slab_at(i);
            uint8_t *sc = score + (keep ? i * nr * kScoreLd : 0);
            if (!keep) {
                cp_async_wait<S - 1>();
                __syncwarp();
                scores(ring + (it % S) * (kSlab * D), j0, sc, false, true);
                issue(it + S);
                ++it;
            }
            // probabilities in place of the scores: the row's first 32 bytes
            uint32_t there;
            const bool plain = plain_slab(j0, there);
            for (int k = 0; k < nr; ++k) {
                const int32_t rm = __shfl_sync(0xffffffffu, xm, k);
                const int32_t x = *reinterpret_cast<const int16_t *>(sc + k * kScoreLd + 2 * lane);
                int32_t p = shift_exp_one(x, rm, a.frac_bits);
                if (!plain && !(((there >> lane) & 1) && sees(a, r, (row0 + k) / G, j0 + lane))) p = 0;
                __syncwarp();
                sc[k * kScoreLd + lane] = (uint8_t)p;
            }
            cp_async_wait<S - 1>();
            __syncwarp();
            const uint8_t *vs = ring + (it % S) * (kSlab * D);
            const uint8_t *pr = sc + g * kScoreLd + 4 * t;
            uint32_t a0 = 0, a1 = 0, a2 = 0, a3 = 0;
            if (g < nr) a0 = *reinterpret_cast<const uint32_t *>(pr), a2 = *reinterpret_cast<const uint32_t *>(pr + 16);
            if (g + 8 < nr) {
                a1 = *reinterpret_cast<const uint32_t *>(pr + 8 * kScoreLd);
                a3 = *reinterpret_cast<const uint32_t *>(pr + 8 * kScoreLd + 16);
            }
            sum0 = (int32_t)__dp4a(a0, 0x01010101u, __dp4a(a2, 0x01010101u, (uint32_t)sum0));
            sum1 = (int32_t)__dp4a(a1, 0x01010101u, __dp4a(a3, 0x01010101u, (uint32_t)sum1));
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                uint32_t v[4];
                ldsm_trans_b8(v, vs + lane * D + v_piece<D>(lane, c) * 16);
                mma_u8s8(o[2 * c], a0, a1, a2, a3, v[0], v[2]);
                mma_u8s8(o[2 * c + 1], a0, a1, a2, a3, v[1], v[3]);
            }
            __syncwarp();
            issue(it + S);
            ++it;
        }
        cp_async_wait<0>();
        // sums over the warps, then over the cluster
        sum0 += __shfl_xor_sync(0xffffffffu, sum0, 1);
        sum1 += __shfl_xor_sync(0xffffffffu, sum1, 1);
        sum0 += __shfl_xor_sync(0xffffffffu, sum0, 2);
        sum1 += __shfl_xor_sync(0xffffffffu, sum1, 2);
        if (mine) {
            if (t == 0 && g < nr) atomicAdd(&s_sum[g], sum0);
            if (t == 0 && g + 8 < nr) atomicAdd(&s_sum[g + 8], sum1);
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                int32_t *d = s_o + 8 * i + 2 * t;
                if (g < nr) atomicAdd(d + g * D, o[i][0]), atomicAdd(d + g * D + 1, o[i][1]);
                if (g + 8 < nr) atomicAdd(d + (g + 8) * D, o[i][2]), atomicAdd(d + (g + 8) * D + 1, o[i][3]);
            }
        }
        auto write = [&](auto total) {  // four channels per thread, rows dealt out over the cluster
            for (int i = rank * 32 * kFewWarps + tid; i < nr * (D / 4); i += ranks * 32 * kFewWarps) {
                const int k = i / (D / 4), d = (i % (D / 4)) * 4, row = row0 + k;
                const int32_t inv = fisr(total(s_sum, k), a.rsqrt_offset);
                uint32_t w = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) w |= (uint32_t)(finish(a, total(s_o, k * D + d + e), inv) & 255) << (8 * e);
                *reinterpret_cast<uint32_t *>(a.y + (int64_t)(r.first + row / G) * a.ldy +
                                              (int64_t)(kvh * G + row % G) * D + d) = w;
            }
        };
        if (ranks == 1) {
            __syncthreads();
            write([&](int32_t *p, int i) { return p[i]; });
            __syncthreads();
        } else {
            cg::cluster_group cl = cg::this_cluster();
            cl.sync();
            write([&](int32_t *p, int i) {
                uint32_t v = 0;
                for (int k = 0; k < ranks; ++k) v += (uint32_t)cl.map_shared_rank(p, k)[i];
                return (int32_t)v;
            });
            cl.sync();  // no block's sums go away or are cleared while another reads them
        }
    }
}

template <int D>
static cudaError_t few_rows(const TreeAttnArgs &a, cudaStream_t st) {
    const int64_t keys = std::max<int64_t>(1, (int64_t)a.width << a.page_log2), pairs = (int64_t)a.B * a.Hkv;
    // split the keys while the pairs alone leave SMs idle and a block keeps 256
    // keys, or while a block would have more than 4096
    int ranks = 1;
    while (ranks < 8 && ((pairs * ranks < 3 * num_sms() && keys / ranks > 256) || keys / ranks > 4096)) ranks *= 2;
    const int64_t per_warp = (keys / kSlab / ranks + kFewWarps) / kFewWarps;
    const int64_t guess = std::min<int64_t>(16, std::max<int64_t>(1, (a.N + a.B - 1) / a.B * (a.H / a.Hkv)));
    const int cap = (int)std::min<int64_t>(12 * 1024, std::max<int64_t>(16 * kScoreLd, per_warp * guess * kScoreLd));
    const size_t smem = Few<D>::smem(cap);
    static SmemLimit lim;
    cudaError_t e = raise_smem_limit(few_rows_kernel<D>, smem, lim);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ranks, a.Hkv, a.B);
    cfg.blockDim = dim3(32 * kFewWarps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, few_rows_kernel<D>, a, cap);
}

}  // namespace tree

cudaError_t tree_attention(const TreeAttnArgs &a, cudaStream_t st) {
    if (a.B == 0) return cudaMemset2DAsync(a.y, a.ldy, 0, (size_t)a.H * a.D, (size_t)a.N, st);
    return a.D == 64 ? tree::few_rows<64>(a, st) : tree::few_rows<128>(a, st);
}

}  // namespace iw
