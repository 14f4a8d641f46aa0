// tree_attn.cu -- integer attention of ragged drafted trees over a paged INT8
// cache (iw_tree_attention). With x = sat16(rrs(q.k * m, s)) for the keys that
// a row sees and M their maximum,
//   p = shift_exp(x - M - 1),  o = clamp(rrs(rrs(rrs(sum p v * i, f) * i, f) * am, as)),
//   i = fisr(sum p)  with f = rsqrt_offset,
// the steps of the dense attention (kernels.cu). All sums are integers, so how
// the keys are split does not change a bit of the result.
#include <cooperative_groups.h>

#include "iw_common.cuh"
#include "iw_sm100.cuh"
#include "iw_tmap.cuh"
#include "paged.cuh"

namespace iw {
namespace tree {

// Keys per step of a warp: 4 KB of K or V.
template <int D>
struct Slab {
    static constexpr int kKeys = 4096 / D;
};

// c += a (16 rows x 32, signed bytes) * b (32 x 8 bytes, signed or unsigned).
// Lane (g = lane/4, t = lane%4) holds a0/a1: rows g/g+8, k 4t..4t+3, a2/a3:
// the same rows, k 16+4t..; b0/b1: column g, k 4t.. / 16+4t..; c0,c1/c2,c3:
// rows g/g+8, columns 2t, 2t+1.
IW_DEV void mma_s8(int32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
IW_DEV void mma_s8u8(int32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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

// Raw scores of a slab: accumulators of its 16-key tiles.
template <int D>
struct Scores {
    int32_t c[Slab<D>::kKeys / 16][4];
};

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

// Byte offset of row j of a page within the caches' head.
IW_DEV uint64_t row_at(const TreeAttnArgs &a, int32_t page, int j) {
    return (uint64_t)(uint32_t)page * a.page_stride + (uint64_t)((uint32_t)j & ((1u << a.page_log2) - 1)) * a.row_stride;
}
IW_DEV bool has_page(const TreeAttnArgs &a, const Request &r, int j) {
    return j < r.keys && (uint32_t)r.table[j >> a.page_log2] < a.n_pages;
}

// (x - M - 1) -> the probability, x <= M the requantised score: shift_exp_one
// by fewer steps where the exponent's fraction has 7 to 14 bits. With
// d = x - M - 1 in [-65536, -1]: the 16-bit steps of the definition wrap where
// d < -22795, which then gives 0 (a positive exponent), and d = -65536 wraps to 0,
// the largest probability.
struct ExpK {
    int32_t fb, one, mask, sh;
    bool quick;
};
IW_DEV ExpK exp_k(int32_t fb) { return {fb, 1 << (fb & 15), (1 << (fb & 15)) - 1, fb - 7, fb >= 7 && fb <= 14}; }
IW_DEV int32_t quick_exp(int32_t d, const ExpK &k) {
    const int32_t f = d + (d >> 1) - (d >> 4);
    const uint32_t num = (uint32_t)(((f & k.mask) >> 1) + k.one);
    int32_t p;
    asm("shr.u32 %0, %1, %2;" : "=r"(p) : "r"(num), "r"(k.sh - (f >> k.fb)));  // 0 for shifts above 31
    if (d < -22795) p = d == -65536 ? 128 : 0;
    return p;
}

// The normalisation of one output channel.
struct FinishK {
    RrsK norm, out;
    int32_t av_mult;
};
IW_DEV int32_t finish(const FinishK &k, int32_t acc, int32_t inv) {
    int32_t v = rrs_apply(wmul(acc, inv), k.norm);
    v = rrs_apply(wmul(v, inv), k.norm);
    return clampi(rrs_apply(wmul(v, k.av_mult), k.out), -127, 127);
}

// Rows from starts[B] on are padding: the blocks of the last request zero
// them, each its own heads.
IW_DEV void zero_padding(const TreeAttnArgs &a, int kvh, int rank, int ranks) {
    const int64_t first = max(a.starts[a.B], 0);
    const int G = a.G, per = G * a.D / 16;
    for (int64_t i = (int64_t)rank * blockDim.x + threadIdx.x; i < (a.N - first) * per; i += (int64_t)ranks * blockDim.x)
        *reinterpret_cast<int4 *>(a.y + (first + i / per) * a.ldy + (int64_t)kvh * G * a.D + (i % per) * 16) =
            make_int4(0, 0, 0, 0);
}

// 16-byte piece c of row `row` of a slab in shared memory lies at piece
// swz(row, c): the 64- and 128-byte swizzles of the tensor maps, under which 8
// consecutive rows have one piece in different banks.
template <int D>
IW_DEV int swz(int row, int c) { return D == 64 ? c ^ ((row >> 1) & 3) : c ^ (row & 7); }

// Loading a slab of keys of one head, completing on `bar`. TMA: one box per page
// (or slab's worth of one) through the cache's tensor map, lane i the i-th;
// pages of fewer than 8 rows do not fill a swizzle pattern and go by 16-byte
// cp.async instead. Rows without a page, or past the last key's, are left as
// they are: whatever is there is masked.
template <int D>
IW_DEV void load_boxes(const TreeAttnArgs &a, const CUtensorMap *map, int kvh, int j0, int box, int32_t page, bool ok,
                       uint8_t *dst, uint64_t *bar) {
    const int lane = threadIdx.x & 31;
    const uint32_t n = __popc(__ballot_sync(0xffffffffu, ok));
    if (lane == 0) mbar_arrive_expect_tx(bar, n * box * D);
    __syncwarp();
    if (ok)
        tma_load_4d(map, bar, dst + lane * box * D, 0, (j0 + lane * box) & ((1 << a.page_log2) - 1), kvh, page);
}
template <int D>
IW_DEV void load_rows(const TreeAttnArgs &a, const Request &r, const int8_t *head, int j0, uint8_t *dst, uint64_t *bar) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int row = (e * 32 + lane) / (D / 16), c = lane % (D / 16), j = j0 + row;
        if (has_page(a, r, j))
            cp_async16(dst + row * D + swz<D>(row, c) * 16, head + row_at(a, r.table[j >> a.page_log2], j) + 16 * c);
    }
    mbar_arrive_cp_async(bar);
}
// Bounded wait for a slab; a wait that gives up sets the device status word.
IW_DEV void slab_wait(uint64_t *bar, uint32_t parity) {
    uint64_t t0 = 0;
    for (uint32_t i = 1; !mbar_try_wait_suspend(bar, parity, 200000u); ++i)
        if ((i & 63u) == 0) {
            if (t0 == 0) t0 = globaltimer_ns();
            else if (globaltimer_ns() - t0 > g_wait_timeout_ns) {
                atomicOr(&g_device_status, IW_DEVERR_WAIT_TIMEOUT);
                break;
            }
        }
    __syncwarp();
}

// ---------------------------------------------------------------------------
// Few rows per key head (single tokens, small trees): bound by reading K and V
// once from HBM. Blocks of one to four warps, or a cluster of them, serve one
// (request, key head) and split its keys; each warp streams slabs of 4 KB
// through a ring of its own (TMA, no block barrier), K first: scores of the
// slab's keys by 8 rows by mma.sync with the keys as the 16-row operand, the raw scores kept in
// shared memory so that K is not read again once the maximum over all
// blocks is known (exchanged through distributed shared memory; the
// requantisation is monotone, so the maximum is taken of raw scores); then V:
// probabilities, one thread per (row, key), and (P.V)^T by mma.sync with V
// transposed by ldmatrix. mma.sync and not tcgen05: with at most 8 rows the
// 128-row tile would be padding, and the tensor pipe is far from its limit at
// HBM rate; what counts is the instructions per slab.
// ---------------------------------------------------------------------------
constexpr int kFewRows = 8;

// D: head dimension, W: warps per block, NR: most rows at a time (1 or 8)
template <int D, int W, int NR>
struct Few {
    static constexpr int kStages = 2;
    static constexpr int kRing = kStages * 4096;
    static constexpr int kScoreLd = Slab<D>::kKeys + 4;  // words per row of a slab's raw scores, padded against bank conflicts
    static constexpr int kOutLd = D + 4;
    static size_t smem(int slots) {
        return 1024 + (size_t)W * (kRing + kStages * 8 + slots * kScoreLd * 4) + (NR * kOutLd + 2 * NR) * 4;
    }
};

// Grid: x = ranks * row blocks, y = key heads, z = requests. A row block takes
// every (row blocks)-th group of `group` rows.
template <int D, int W, int NR, bool TMA>
__global__ void __launch_bounds__(32 * W, (D == 64 ? 20 : 12) / W)
    few_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                    TreeAttnArgs a, int ranks, int group, int slots) {
    namespace cg = cooperative_groups;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_align1024(smem_raw);
    using F = Few<D, W, NR>;
    constexpr int S = F::kStages, OLD = F::kOutLd, SL = Slab<D>::kKeys, kScoreLd = F::kScoreLd;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    uint8_t *ring = smem + warp * F::kRing;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + W * F::kRing) + warp * S;
    int32_t *scores = reinterpret_cast<int32_t *>(smem + W * (F::kRing + S * 8));
    int32_t *score = scores + warp * slots * kScoreLd, *s_o = scores + W * slots * kScoreLd;
    int32_t *s_sum = s_o + NR * OLD, *s_max = s_sum + NR;
    const int lr = 31 - __clz(ranks);  // a power of two
    const int rank = blockIdx.x & (ranks - 1), kvh = blockIdx.y, b = blockIdx.z, G = a.G;
    if (lane < S) mbar_init(&bars[lane], TMA ? 1 : 32);
    fence_mbar_init();
    if (TMA && tid == 0) prefetch_tmap(&tmap_k), prefetch_tmap(&tmap_v);
    __syncwarp();
    pdl_wait();
    pdl_launch();
    if (b == a.B - 1) zero_padding(a, kvh, blockIdx.x, gridDim.x);
    const Request r = request(a, b);
    const int rows = r.fresh * G, first_row = (int)(blockIdx.x >> lr) * group, row_step = (int)(gridDim.x >> lr) * group;
    if (first_row >= rows) return;
    const int8_t *kbase = a.k + kvh * a.head_stride, *vbase = a.v + kvh * a.head_stride;
    // this block's slabs, then this warp's
    const int slabs = (r.keys + SL - 1) / SL;
    const int first = (slabs * rank) >> lr, count = ((slabs * (rank + 1)) >> lr) - first;
    const int slab0 = first + count * warp / W, mine = first + count * (warp + 1) / W - slab0;
    // pages in boxes of at most a slab's rows; lane i holds the page of box i of a
    // window of 32 boxes, -1 for one that has no page
    const int box = min(1 << a.page_log2, SL), per = SL / box;
    int32_t pages = -1;
    bool holes = false;  // keys of this warp without a page
    auto window = [&](int i) {
        const int j = (slab0 + i) * SL + lane * box;
        const bool real = j < min((slab0 + mine) * SL, r.keys);
        pages = real ? r.table[j >> a.page_log2] : -1;
        if ((uint32_t)pages >= a.n_pages) pages = -1;
        holes |= real && pages < 0;
    };
    if (TMA) {
        const int span = 32 / per;
        for (int i = mine > 0 ? (mine - 1) & -span : -1; i >= 0; i -= span) window(i);
    } else {
        for (int j = slab0 * SL + lane; j < min((slab0 + mine) * SL, r.keys); j += 32) holes |= !has_page(a, r, j);
    }
    holes = __any_sync(0xffffffffu, holes);
    const int all_see = holes ? 0 : min(r.ctx, r.keys);  // keys below are seen by every row
    auto token = [&](int row) { return G == 1 ? row : row / G; };
    const RrsK rk = rrs_k(a.qk_shift);
    const ExpK ek = exp_k(a.frac_bits);
    const FinishK fk{rrs_k(a.rsqrt_offset), rrs_k(a.av_shift), a.av_mult};
    auto requant = [&](int32_t acc) { return clampi(rrs_apply(wmul(acc, a.qk_mult), rk), -32768, 32767); };

    uint32_t base = 0;  // slabs streamed for earlier rows
    for (int row0 = first_row; row0 < rows; row0 += row_step, base += 2 * mine) {
        const int nr = NR == 1 ? 1 : min(group, rows - row0);
        const bool keep = mine * nr <= slots;  // otherwise the second pass computes the scores again
        auto issue = [&](int it) {             // the stream of slabs: K0 .. Kn-1, V0 .. Vn-1
            if (it >= 2 * mine) return;
            const bool v = it >= mine;
            const int i = v ? it - mine : it, j0 = (slab0 + i) * SL, slot = (base + it) % S;
            if (TMA) {
                const int at = (i * per) & 31;
                if (at == 0 && mine * per > 32) window(i);
                const int32_t page = __shfl_sync(0xffffffffu, pages, (at + lane) & 31);
                load_boxes<D>(a, v ? &tmap_v : &tmap_k, kvh, j0, box, page, lane < per && page >= 0, ring + slot * 4096,
                              &bars[slot]);
            } else {
                load_rows<D>(a, r, v ? vbase : kbase, j0, ring + slot * 4096, &bars[slot]);
            }
        };
        auto arrived = [&](int it) -> const uint8_t * {
            const int slot = (base + it) % S;
            slab_wait(&bars[slot], ((base + it) / S) & 1);
            return ring + slot * 4096;
        };
#pragma unroll 1
        for (int i = 0; i < S; ++i) issue(i);

        // queries: lane's 16 bytes of row g in each 64-byte half, so that bytes
        // 8s.. and 8s+4.. of a piece are the two registers of step s (the same
        // order of channels as in the keys' pieces below)
        int4 q[D / 64];
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
            q[c] = make_int4(0, 0, 0, 0);
            const int row = row0 + g, n = token(row);
            if (g < nr)
                q[c] = *reinterpret_cast<const int4 *>(a.q + (int64_t)(r.first + n) * a.ldq +
                                                       (int64_t)(kvh * G + row - n * G) * a.q_hs + 64 * c + 16 * t);
        }
        if (W > 1) {
            for (int i = tid; i < NR * OLD + 2 * NR; i += 32 * W) s_o[i] = i < NR * OLD + NR ? 0 : INT32_MIN;
            __syncthreads();
        }
        // which of the lane's keys j0 + 32e + lane the rows see, for a slab that is
        // not seen whole
        auto seen = [&](int k, int j) {
            const int u = j - r.ctx;
            if (j >= r.keys || (holes && !has_page(a, r, j))) return false;
            if (u < 0) return true;
            const int n = token(row0 + k);
            if (a.words == 0) return u <= n;
            return (u >> 5) < a.words && ((a.mask[(int64_t)(r.first + n) * a.words + (u >> 5)] >> (u & 31)) & 1);
        };
        int32_t m0 = INT32_MIN, m1 = INT32_MIN, mr = INT32_MIN;  // rows 2t, 2t+1 (own keys); row = lane (other slabs)
        // the key of a lane's fragment rows: a quarter warp reads two rows, of 64
        // bytes each, that must not share banks: rows g and g+1 of 64 bytes, rows
        // that differ in bit 2 of 128 (swizzled) bytes
        const int gk = D == 64 ? g : (g >> 1) | ((g & 1) << 2);
        // raw scores of the keys 16m + gk and 16m + 8 + gk with all rows; load(row, h)
        // gives the lane's piece of a key's half h
        auto raw = [&](Scores<D> &x, auto load) {
            auto &c = x.c;
#pragma unroll
            for (int m16 = 0; m16 < SL / 16; ++m16) {
                c[m16][0] = c[m16][1] = c[m16][2] = c[m16][3] = 0;
#pragma unroll
                for (int h = 0; h < D / 64; ++h) {
                    const int4 ka = load(16 * m16 + gk, h), kb = load(16 * m16 + 8 + gk, h);
                    mma_s8(c[m16], ka.x, kb.x, ka.y, kb.y, q[h].x, q[h].y);
                    mma_s8(c[m16], ka.z, kb.z, ka.w, kb.w, q[h].z, q[h].w);
                }
            }
        };
        auto store = [&](int32_t *to, const Scores<D> &x) {
            auto &c = x.c;
            int32_t *w = to + 2 * t * kScoreLd + gk;
            if (2 * t < nr) {
#pragma unroll
                for (int m = 0; m < SL / 16; ++m) w[16 * m] = c[m][0], w[16 * m + 8] = c[m][2];
            }
            if (NR > 1 && 2 * t + 1 < nr) {
                w += kScoreLd;
#pragma unroll
                for (int m = 0; m < SL / 16; ++m) w[16 * m] = c[m][1], w[16 * m + 8] = c[m][3];
            }
        };
        int it = 0;
#pragma unroll 1
        for (; it < mine; ++it) {
            const int j0 = (slab0 + it) * SL;
            const uint8_t *ks = arrived(it);
            Scores<D> x;
            raw(x, [&](int row, int h) {
                return *reinterpret_cast<const int4 *>(ks + row * D + swz<D>(row, 4 * h + t) * 16);
            });
            __syncwarp();
            issue(it + S);
            const bool plain = j0 + SL <= all_see;
            int32_t *to = score + (keep ? it * nr * kScoreLd : 0);
            if (keep || !plain) store(to, x);
            if (plain) {
#pragma unroll
                for (int m = 0; m < SL / 16; ++m) {
                    m0 = max(m0, max(x.c[m][0], x.c[m][2]));
                    if (NR > 1) m1 = max(m1, max(x.c[m][1], x.c[m][3]));
                }
            } else {
                __syncwarp();
#pragma unroll 1
                for (int k = 0; k < nr; ++k) {
                    int32_t m = INT32_MIN;
#pragma unroll
                    for (int e = 0; e < SL; e += 32)
                        if (seen(k, j0 + e + lane)) m = max(m, to[k * kScoreLd + e + lane]);
                    m = __reduce_max_sync(0xffffffffu, m);
                    if (lane == k) mr = max(mr, m);
                }
                __syncwarp();
            }
        }
        // row maxima: over the lanes, the warps, the cluster
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            m0 = max(m0, __shfl_xor_sync(0xffffffffu, m0, o));
            if (NR > 1) m1 = max(m1, __shfl_xor_sync(0xffffffffu, m1, o));
        }
        int32_t xm;  // row = lane
        if (W == 1) {
            xm = __shfl_sync(0xffffffffu, m0, (lane >> 1) & 3);
            if (NR > 1) {
                const int32_t odd = __shfl_sync(0xffffffffu, m1, (lane >> 1) & 3);
                if (lane & 1) xm = odd;
            }
            xm = max(xm, mr);
        } else {
            if (g == 0 && 2 * t < NR) atomicMax(&s_max[2 * t], m0);
            if (g == 0 && 2 * t + 1 < NR) atomicMax(&s_max[2 * t + 1], m1);
            if (lane < nr && mr != INT32_MIN) atomicMax(&s_max[lane], mr);
            if (ranks == 1) {
                __syncthreads();
                xm = s_max[lane & (NR - 1)];
            } else {
                cg::cluster_group cl = cg::this_cluster();
                cl.sync();
                xm = INT32_MIN;
                for (int k = 0; k < ranks; ++k) xm = max(xm, cl.map_shared_rank(s_max, k)[lane & (NR - 1)]);
            }
        }
        xm = (xm == INT32_MIN ? -32768 : requant(xm)) + 1;

        int32_t o[D / 16][4];  // channels 16i + g (and + 8) of rows 2t, 2t+1
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0;
        uint32_t sum = 0;  // row g, own keys
#pragma unroll 1
        for (; it < 2 * mine; ++it) {
            const int i = it - mine, j0 = (slab0 + i) * SL;
            int32_t *sc = score + (keep ? i * nr * kScoreLd : 0);
            if (!keep) {
                Scores<D> x;
                raw(x, [&](int row, int h) {
                    const int j = min(j0 + row, r.keys - 1);
                    const int32_t page = r.table[j >> a.page_log2];
                    if (holes && (uint32_t)page >= a.n_pages) return make_int4(0, 0, 0, 0);
                    return *reinterpret_cast<const int4 *>(kbase + row_at(a, page, j) + 64 * h + 16 * t);
                });
                store(sc, x);
            }
            __syncwarp();
            // probabilities in place of the scores: the first bytes of the row
            const bool plain = j0 + SL <= all_see;
#pragma unroll 1
            for (int k = 0; k < nr; ++k) {
                const int32_t rm = __shfl_sync(0xffffffffu, xm, k);
                int32_t p[SL / 32];
#pragma unroll
                for (int e = 0; e < SL / 32; ++e) {
                    const int32_t x = requant(sc[k * kScoreLd + 32 * e + lane]);
                    p[e] = ek.quick ? quick_exp(x - rm, ek) : shift_exp_one(x, (int16_t)rm, a.frac_bits);
                }
                if (!plain) {
#pragma unroll
                    for (int e = 0; e < SL / 32; ++e)
                        if (!seen(k, j0 + 32 * e + lane)) p[e] = 0;
                }
                __syncwarp();
#pragma unroll
                for (int e = 0; e < SL / 32; ++e) reinterpret_cast<uint8_t *>(sc + k * kScoreLd)[32 * e + lane] = (uint8_t)p[e];
            }
            __syncwarp();
            uint32_t p[SL / 16];
#pragma unroll
            for (int e = 0; e < SL / 16; ++e) {
                p[e] = g < nr ? sc[g * kScoreLd + 4 * e + t] : 0;
                sum = __dp4a(p[e], 0x01010101u, sum);
            }
            const uint8_t *vs = arrived(it);
#pragma unroll
            for (int c = 0; c < D / 16; ++c)
#pragma unroll
                for (int e = 0; e < SL / 32; ++e) {
                    const int row = 32 * e + lane;
                    uint32_t v[4];
                    ldsm_trans_b8(v, vs + row * D + swz<D>(row, c) * 16);
                    mma_s8u8(o[c], v[0], v[1], v[2], v[3], p[2 * e], p[2 * e + 1]);
                }
            __syncwarp();
            issue(it + S);
        }
        // sums over the warps, then over the cluster
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        auto give = [&](int32_t *d, int32_t v) {
            if (W > 1) atomicAdd(d, v);
            else *d = v;
        };
        if (W == 1 || mine) {
            if (t == 0 && g < nr) give(&s_sum[g], (int32_t)sum);
            int32_t *d = s_o + 2 * t * OLD + g;
            if (2 * t < nr) {
#pragma unroll
                for (int c = 0; c < D / 16; ++c) give(d + 16 * c, o[c][0]), give(d + 16 * c + 8, o[c][2]);
            }
            if (NR > 1 && 2 * t + 1 < nr) {
#pragma unroll
                for (int c = 0; c < D / 16; ++c) give(d + OLD + 16 * c, o[c][1]), give(d + OLD + 16 * c + 8, o[c][3]);
            }
        }
        auto write = [&](auto total) {  // two channels per thread, dealt out over the cluster
            int32_t inv = 0;            // row = lane
            if (lane < nr) inv = fisr(total(s_sum, lane), a.rsqrt_offset);
#pragma unroll 1
            for (int i0 = (rank * W + warp) * 32; i0 < nr * (D / 2); i0 += ranks * W * 32) {
                const int i = i0 + lane, k = i0 / (D / 2), d = (i % (D / 2)) * 2, row = row0 + k, n = token(row);
                const int32_t v = __shfl_sync(0xffffffffu, inv, k);
                char2 w;
                w.x = (signed char)finish(fk, total(s_o, k * OLD + d), v);
                w.y = (signed char)finish(fk, total(s_o, k * OLD + d + 1), v);
                *reinterpret_cast<char2 *>(a.y + (int64_t)(r.first + n) * a.ldy + (int64_t)(kvh * G + row - n * G) * D + d) = w;
            }
        };
        if (ranks == 1) {
            if (W > 1) __syncthreads();
            else __syncwarp();
            write([&](int32_t *p, int i) { return p[i]; });
            if (W > 1) __syncthreads();
            else __syncwarp();
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

// Kernel launch with clusters of `ranks` blocks along x and the PDL attribute.
template <typename... KArgs, typename... Args>
static cudaError_t launch_cluster(void (*kernel)(KArgs...), int ranks, dim3 grid, dim3 block, size_t smem,
                                  cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ranks > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Tensor maps of the caches: boxes of one head's rows of one page.
struct CacheMaps {
    CUtensorMap k, v;
};
static cudaError_t cache_maps(const TreeAttnArgs &a, CacheMaps &m) {
    const uint64_t sizes[4] = {(uint64_t)a.D, 1ull << a.page_log2, (uint64_t)a.Hkv, a.n_pages};
    const uint64_t strides[3] = {a.row_stride, (uint64_t)a.head_stride, a.page_stride};
    const uint32_t box[4] = {(uint32_t)a.D, std::min(1u << a.page_log2, 4096u / a.D), 1, 1};
    const CUtensorMapSwizzle swz = a.D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    cudaError_t e = make_tmap_4d_u8(&m.k, a.k, sizes, strides, box, swz);
    return e == cudaSuccess ? make_tmap_4d_u8(&m.v, a.v, sizes, strides, box, swz) : e;
}

// How the few-rows kernel is cut: warps per block, blocks per cluster, rows at a
// time, row blocks, score slots per warp.
struct FewPlan {
    int warps, ranks, group, row_blocks, slots;
};

template <int D, int W, int NR, bool TMA>
static cudaError_t few_rows_launch(const TreeAttnArgs &a, const CacheMaps &m, const FewPlan &p, cudaStream_t st) {
    const size_t smem = Few<D, W, NR>::smem(p.slots);
    static SmemLimit lim;
    cudaError_t e = raise_smem_limit(few_rows_kernel<D, W, NR, TMA>, smem, lim);
    if (e != cudaSuccess) return e;
    return launch_cluster(few_rows_kernel<D, W, NR, TMA>, p.ranks, dim3(p.ranks * p.row_blocks, a.Hkv, a.B), dim3(32 * W),
                          smem, st, m.k, m.v, a, p.ranks, p.group, p.slots);
}

template <int D, int NR>
static cudaError_t few_rows_warps(const TreeAttnArgs &a, const CacheMaps &m, bool tma, const FewPlan &p, cudaStream_t st) {
    if (!tma) return few_rows_launch<D, 4, NR, false>(a, m, p, st);
    if (p.warps == 1) return few_rows_launch<D, 1, NR, true>(a, m, p, st);
    if (p.warps == 2) return few_rows_launch<D, 2, NR, true>(a, m, p, st);
    return few_rows_launch<D, 4, NR, true>(a, m, p, st);
}

template <int D>
static cudaError_t few_rows(const TreeAttnArgs &a, const CacheMaps &m, bool tma, int64_t mean_rows, cudaStream_t st) {
    const int64_t keys = std::max<int64_t>(1, (int64_t)a.width << a.page_log2), pairs = (int64_t)a.B * a.Hkv;
    FewPlan p{tma ? 1 : 4, 1, kFewRows, 1, 0};
    // One warp per (request, key head) needs no barrier and shares no sums; more
    // warps, then more blocks, while the SMs have fewer than 16 warps each and a
    // warp keeps 64 keys, or while a warp would have more than 1024
    while (p.warps * p.ranks < 32) {
        const int64_t share = keys / (p.warps * p.ranks);
        if (!((pairs * p.warps * p.ranks < 16 * (int64_t)num_sms() && share > 64) || share > 1024)) break;
        if (p.warps < 4) p.warps *= 2;
        else p.ranks *= 2;
    }
    // fewer rows at a time while the SMs have fewer than 4 warps each: a warp's
    // time goes by its rows
    const int64_t guess = std::min<int64_t>(kFewRows, mean_rows);
    while (p.group > 1 && (p.group >= 2 * guess || pairs * p.warps * p.ranks * ((guess + p.group - 1) / p.group) < 4 * num_sms()))
        p.group /= 2;
    p.row_blocks = (int)((guess + p.group - 1) / p.group);
    // room for the scores of every slab
    const int64_t per_warp = (keys / Slab<D>::kKeys / p.ranks + p.warps) / p.warps;
    p.slots = (int)std::min<int64_t>(64, std::max<int64_t>(1, per_warp) * p.group);
    return p.group == 1 ? few_rows_warps<D, 1>(a, m, tma, p, st) : few_rows_warps<D, kFewRows>(a, m, tma, p, st);
}

}  // namespace tree

cudaError_t tree_attention(const TreeAttnArgs &a, cudaStream_t st) {
    if (a.B == 0) return cudaMemset2DAsync(a.y, a.ldy, 0, (size_t)a.H * a.D, (size_t)a.N, st);
    // tensor maps need pages of 8 rows or more and axes that step
    const bool tma = a.page_log2 >= 3 && a.n_pages > 0 && a.row_stride > 0 && a.head_stride > 0 && a.page_stride > 0;
    tree::CacheMaps m = {};
    if (tma)
        if (cudaError_t e = tree::cache_maps(a, m); e != cudaSuccess) return e;
    const int64_t mean_rows = (a.N + a.B - 1) / a.B * a.G;
    return a.D == 64 ? tree::few_rows<64>(a, m, tma, mean_rows, st) : tree::few_rows<128>(a, m, tma, mean_rows, st);
}

}  // namespace iw
