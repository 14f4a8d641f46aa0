// tree_attn.cu -- integer attention of ragged drafted trees over a paged INT8
// cache (iw_tree_attention). With x = sat16(rrs(q.k * m, s)) for the keys that
// a row sees and M their maximum,
//   p = shift_exp(x - M - 1),  o = clamp(rrs(rrs(rrs(sum p v * i, f) * i, f) * am, as)),
//   i = fisr(sum p)  with f = rsqrt_offset,
// the steps of the dense attention (kernels.cu). All sums are integers, so how
// the keys are split does not change a bit of the result.
#include <cooperative_groups.h>

#include <type_traits>

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

// c += a (16 rows x 32 bytes) * b (32 x 8 bytes), either signed or unsigned.
// Lane (g = lane/4, t = lane%4) holds a0/a1: rows g/g+8, k 4t..4t+3, a2/a3:
// the same rows, k 16+4t..; b0/b1: column g, k 4t.. / 16+4t..; c0,c1/c2,c3:
// rows g/g+8, columns 2t, 2t+1.
IW_DEV void mma_s8(int32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
IW_DEV void mma_s8u8(int32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// c = a * b, signed.
IW_DEV void mma_s8_first(int32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
// Two 16 x 16 byte tiles, transposed: lanes 0-15 point at the rows of the
// first, 16-31 at those of the second; r0/r1: rows 4t..4t+3 of columns g / 8+g
// of the first tile, r2/r3 of the second.
IW_DEV void ldsm_trans_b8(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
}
IW_DEV int4 lds_v4(uint32_t at) {
    int4 v;
    asm volatile("ld.shared.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
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

// The request that block row z serves: of up to 32 long requests the z-th by
// decreasing work, so that the last blocks to start are not the longest (16
// requests of 1000 to 8191 keys and 24 to 64 tokens on 4 x 8 heads, the longest
// given last: 355 us in the given order, 321 so).
IW_DEV int pick_request(const TreeAttnArgs &a, int z) {
    if (!a.largest_first) return z;
    const int lane = threadIdx.x & 31;
    int64_t work = -1;
    if (lane < a.B) {
        const int64_t fresh = max(a.starts[lane + 1] - a.starts[lane], 0);
        work = fresh ? (max(a.ctx[lane], 0) + fresh) * ((fresh * a.G + 15) / 16) : 0;
    }
    int before = 0;
    for (int j = 0; j < a.B; ++j) {
        const int64_t other = __shfl_sync(0xffffffffu, work, j);
        before += other > work || (other == work && j < lane);
    }
    return __ffs(__ballot_sync(0xffffffffu, lane < a.B && before == z)) - 1;
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

// Maximum or sum over the cluster's blocks of one value or four of their shared
// memory, four blocks' loads in flight at a time (a load from another block
// takes hundreds of cycles). A rank count of 1, 2, 4 or 8.
IW_DEV int32_t cluster_max(cooperative_groups::cluster_group cl, int32_t *p, int ranks) {
    int32_t m = INT32_MIN;
    for (int k0 = 0; k0 < ranks; k0 += 4) {
        int32_t v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = *cl.map_shared_rank(p, (k0 + k) & (ranks - 1));
        m = max(max(m, max(v[0], v[1])), max(v[2], v[3]));
    }
    return m;
}
IW_DEV int32_t cluster_sum(cooperative_groups::cluster_group cl, int32_t *p, int ranks) {
    int32_t sum = 0;
    for (int k0 = 0; k0 < ranks; k0 += 4) {
        int32_t v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = *cl.map_shared_rank(p, (k0 + k) & (ranks - 1));
#pragma unroll
        for (int k = 0; k < 4; ++k) sum += k0 + k < ranks ? v[k] : 0;
    }
    return sum;
}
IW_DEV int4 cluster_sum4(cooperative_groups::cluster_group cl, int32_t *p, int ranks) {
    int4 sum = make_int4(0, 0, 0, 0);
    for (int k0 = 0; k0 < ranks; k0 += 4) {
        int4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            v[k] = *reinterpret_cast<const int4 *>(cl.map_shared_rank(p, (k0 + k) & (ranks - 1)));
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k0 + k < ranks) sum.x += v[k].x, sum.y += v[k].y, sum.z += v[k].z, sum.w += v[k].w;
    }
    return sum;
}
// Four channels normalised, as bytes.
IW_DEV uint32_t finish4(const FinishK &k, int4 v, int32_t inv) {
    return (uint32_t)(finish(k, v.x, inv) & 255) | (uint32_t)(finish(k, v.y, inv) & 255) << 8 |
           (uint32_t)(finish(k, v.z, inv) & 255) << 16 | (uint32_t)(finish(k, v.w, inv) & 255) << 24;
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
template <int D, int BYTES>
IW_DEV void load_rows(const TreeAttnArgs &a, const Request &r, const int8_t *head, int j0, uint8_t *dst) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int e = 0; e < BYTES / 512; ++e) {
        const int row = (e * 32 + lane) / (D / 16), c = lane % (D / 16), j = j0 + row;
        if (has_page(a, r, j))
            cp_async16(dst + row * D + swz<D>(row, c) * 16, head + row_at(a, r.table[j >> a.page_log2], j) + 16 * c);
    }
}
// Bounded wait of a warp for a slab. A wait that gives up sets the device
// status word, and this warp's later waits then give up after a millisecond each,
// so that the kernel ends soon and with its copies landed.
struct SlabWait {
    bool late = false;
    IW_DEV void operator()(uint64_t *bar, uint32_t parity) {
        uint64_t t0 = 0;
        for (uint32_t i = 1; !mbar_try_wait_suspend(bar, parity, 200000u); ++i)
            if ((i & 63u) == 0) {
                if (t0 == 0) {
                    t0 = globaltimer_ns();
                } else if (globaltimer_ns() - t0 > (late ? 1000000ull : g_wait_timeout_ns)) {
                    atomicOr(&g_device_status, IW_DEVERR_WAIT_TIMEOUT);
                    late = true;
                    break;
                }
            }
        __syncwarp();
    }
};

// ---------------------------------------------------------------------------
// Few rows per key head (single tokens, small trees): bound by reading K and V
// once from HBM. Blocks of one to four warps, or a cluster of them, serve one
// (request, key head) and split its keys; each warp streams slabs of 4 KB
// through a ring of its own (TMA, no block barrier), K first: scores of the
// slab's keys by 8 rows by mma.sync with the keys as the 16-row operand, the raw
// scores kept in shared memory so that K is not read again once the maximum
// over all blocks is known (exchanged through distributed shared memory; the
// requantisation is monotone, so the maximum is taken of raw scores); then V:
// probabilities, one thread per (row, key), and (P.V)^T by mma.sync with V
// transposed by ldmatrix. mma.sync and not tcgen05: with at most 8 rows the
// 128-row tile would be padding, and the tensor pipe is far from its limit at
// HBM rate; what counts is the instructions per slab. 256 single tokens over 0 to
// 447 keys, 16 heads of 64: 26 us, 4.7 TB/s; 7 over 4097 to 32700 keys, 20 heads: 64
// us, 5.6 TB/s (2 slabs per ring; 1 measured 29 and 80 us, 3 26 and 81: more leave
// room for fewer warps).
// ---------------------------------------------------------------------------
constexpr int kFewRows = 8;

// D: head dimension, W: warps per block, NR: most rows at a time (1 or 8)
template <int D, int W, int NR>
struct Few {
    static constexpr int kStages = 2;
    static constexpr int kRing = kStages * 4096;
    static constexpr int kScoreLd = Slab<D>::kKeys + 4;  // words per row of a slab's raw scores, padded against bank conflicts
    static constexpr int kOutLd = D + 4;
    // the sums are read 16 bytes at a time
    static_assert((kRing + kStages * 8) % 16 == 0 && kScoreLd % 4 == 0 && kOutLd % 4 == 0, "16-byte rows behind the ring");
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
    const int rank = blockIdx.x & (ranks - 1), kvh = blockIdx.y, G = a.G;
    if (lane < S) mbar_init(&bars[lane], TMA ? 1 : 32);
    fence_mbar_init();
    if (TMA && tid == 0) prefetch_tmap(&tmap_k), prefetch_tmap(&tmap_v);
    __syncwarp();
    pdl_wait();
    pdl_launch();
    if (blockIdx.z == a.B - 1) zero_padding(a, kvh, blockIdx.x, gridDim.x);
    const Request r = request(a, pick_request(a, blockIdx.z));
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

    SlabWait slab_wait;
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
                load_rows<D, 4096>(a, r, v ? vbase : kbase, j0, ring + slot * 4096);
                mbar_arrive_cp_async(&bars[slot]);
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
                xm = cluster_max(cl, s_max + (lane & (NR - 1)), ranks);
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
                    ldsm_trans_b8(v, smem_u32(vs) + row * D + swz<D>(row, c) * 16);
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
        auto write = [&](auto total, auto total4) {  // four channels per thread, dealt out over the cluster
            int32_t inv = 0;                         // row = lane
            if (lane < nr) inv = fisr(total(s_sum + lane), a.rsqrt_offset);
#pragma unroll 1
            for (int i0 = (rank * W + warp) * 32; i0 < nr * (D / 4); i0 += ranks * W * 32) {
                const int i = i0 + lane, k = i / (D / 4), d = (i % (D / 4)) * 4, row = row0 + k, n = token(row);
                const int32_t v = __shfl_sync(0xffffffffu, inv, k & 31);
                if (k < nr)
                    *reinterpret_cast<uint32_t *>(a.y + (int64_t)(r.first + n) * a.ldy + (int64_t)(kvh * G + row - n * G) * D +
                                                  d) = finish4(fk, total4(s_o + k * OLD + d), v);
            }
        };
        if (ranks == 1) {
            if (W > 1) __syncthreads();
            else __syncwarp();
            write([](int32_t *p) { return *p; }, [](int32_t *p) { return *reinterpret_cast<const int4 *>(p); });
            if (W > 1) __syncthreads();
            else __syncwarp();
        } else {
            cg::cluster_group cl = cg::this_cluster();
            cl.sync();
            write([&](int32_t *p) { return cluster_sum(cl, p, ranks); }, [&](int32_t *p) { return cluster_sum4(cl, p, ranks); });
            cl.sync();  // no block's sums go away or are cleared while another reads them
        }
    }
}

// ---------------------------------------------------------------------------
// Many rows per key head (trees, prompts, shared key heads): bound by the
// latency and issue of the integer softmax and the score products. A block, or
// a cluster of them that splits the keys, serves up to 64 rows of one (request, key
// head) at a time; four warps compute, a fifth feeds a ring of K and V slots by
// TMA (a full and an empty barrier per slot). A warp holds 16 rows: scores by
// mma.sync, the keys of a tile in such an order that a thread's four
// probabilities are four consecutive operand bytes of P.V, which therefore never
// leave registers; (P.V)^T by mma.sync with V transposed by ldmatrix. Warps share a
// tile between up to four groups of 16 rows; with fewer groups they divide the
// tiles. The maximum needs all keys before the first probability, so the score
// products are taken twice and K is read twice, the second time from L2, or not
// at all where K and V of the request fit the ring.
// 64 requests with trees of 5 to 32 tokens over 64 to 416 keys, 16 heads of 64:
// 39 us. 16 requests with trees of 24 to 64 tokens over 1000 to 8191 keys, 32 query
// and 8 key heads of 128: 298 us, 0.27 of what mma.sync does in 8 bits (1.09 POPS
// measured). More warps per SM, with fewer registers each or the query
// operands in shared memory, measured 296 to 310 us. tcgen05 would multiply
// faster, but hold the scores in tensor memory, from where the softmax has to
// fetch them; not measured. Trees on one head have too few rows for its 128-row
// tiles, shared key heads (96 to 256 rows in the case above) do not.
// ---------------------------------------------------------------------------
constexpr int kManyWarps = 4;

template <int D>
struct Many {
    static constexpr int kStages = D == 64 ? 16 : 8;
    static constexpr int kBytes = 64 * D;  // 64 keys of K or V, or 32 of K and the same of V
    static constexpr int kOutLd = D + 4;
    // the sums of P.V take the ring's place once the tiles are done with
    static size_t smem() { return 1024 + kStages * (kBytes + 16) + 64 * 2 * 4; }
    static_assert(64 * kOutLd * 4 <= kStages * kBytes && kOutLd % 4 == 0, "the sums fit the ring, rows of 16 bytes");
};

// The probability of a score from its raw sum, mostly in the FMA pipe (the ALU
// pipe issues at half its rate). One wide multiply-add and a shift give
// d = x - M - 1: the multiplier m * 2^22 + 1 adds the sum itself, less than
// 2^22, below the product's last place, which rounds halves away from zero. d
// comes with 12582912 added, so that its bits are also the float
// 1.5 * 2^23 + d; floors of d/2 and d/16 are fused multiply-adds rounded down,
// f = d + floor(d/2) - floor(d/16) is exact, and the bits of
// 2^(7 + xi) * (1 + fr / 2^(fb+1)), f = xi * 2^fb + fr, follow by two integer
// multiply-adds; its whole part is the probability. Valid for 7 to 14
// fraction bits and shifts 1 to 9; without CLAMP for rows whose maximum lies
// inside 16 bits and whose cut-off lies above -32768, so that a key clamped from
// below has no probability either way (a cut-off at -32768 itself has one).
struct FastExp {
    int32_t mult, shift, limit, below, mask, scale, zero, half;
};
constexpr int32_t kBias = 0x4B400000;  // bits of 12582912.0f
IW_DEV FastExp fast_exp(const TreeAttnArgs &a) {
    const int fb = min(max(a.frac_bits, 7), 14);
    FastExp k;
    k.mult = (a.qk_mult << 22) + 1;
    k.shift = 22 + (int)min(a.qk_shift, 9u);
    k.limit = kBias - min(22795, 8 << fb);
    k.below = kBias - (8 << fb);
    k.mask = (1 << fb) - 1;
    k.scale = 1 << (23 - fb);
    k.zero = (int32_t)((134u << 23) - ((uint32_t)kBias << (23 - fb)));
    k.half = -(1 << (22 - fb));
    return k;
}
// A row's addend for maximum + 1 = xm.
IW_DEV int64_t fast_base(int32_t xm, const FastExp &k) {
    return ((int64_t)(kBias - xm) << k.shift) + ((int64_t)1 << (k.shift - 1));
}
// CLAMP: for any row. `low` = kBias - 32768 - xm is where x is clamped below; clamped
// above it is 1 below xm; and the difference of both clamps wraps to 0, the
// largest probability.
template <bool CLAMP>
IW_DEV uint32_t fast_prob(int32_t acc, int64_t base, int32_t low, const FastExp &k) {
    const int64_t t = (int64_t)acc * k.mult + base;
    int32_t d = (int32_t)__funnelshift_r((uint32_t)t, (uint32_t)(t >> 32), k.shift);
    if (CLAMP) {
        d = min(max(d, low), kBias - 1);
        if (d == kBias - 65536) return 128;
    }
    d = d < k.limit ? k.below : d;
    const float x = __int_as_float(d);
    const float f = __fadd_rn(x, __fadd_rn(__fmaf_rd(x, 0.5f, 6291456.f), -__fmaf_rd(x, 0.0625f, 11796480.f)));
    const int32_t bits = __float_as_int(f);
    const int32_t w = (bits & k.mask) * k.half + (bits * k.scale + k.zero);
    return __float_as_uint(__fadd_rz(__int_as_float(w), 8388608.f));
}

template <int D, bool TMA>
__global__ void __launch_bounds__(32 * (kManyWarps + 1), D == 64 ? 3 : 2)
    many_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                     TreeAttnArgs a, int ranks) {
    namespace cg = cooperative_groups;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_align1024(smem_raw);
    using F = Many<D>;
    constexpr int S = F::kStages, OLD = F::kOutLd, kTile = 64;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + S * F::kBytes), *empty = full + S;
    int32_t *s_o = reinterpret_cast<int32_t *>(smem), *s_sum = reinterpret_cast<int32_t *>(empty + S), *s_max = s_sum + 64;
    const int lr = 31 - __clz(ranks);  // a power of two
    const int rank = blockIdx.x & (ranks - 1), kvh = blockIdx.y, G = a.G;
    if (TMA && tid == 0) prefetch_tmap(&tmap_k), prefetch_tmap(&tmap_v);
    pdl_wait();
    pdl_launch();
    if (blockIdx.z == a.B - 1) zero_padding(a, kvh, blockIdx.x, gridDim.x);
    const Request r = request(a, pick_request(a, blockIdx.z));
    const int rows = r.fresh * G;
    // RT groups of 16 rows side by side, KG sets of warps that share out the tiles:
    // set i takes tiles of 64 keys i, i + KG, ... through SG slots of the ring that
    // are its own (a set has to see every phase of the barriers it waits on)
    const int lrt = rows <= 16 ? 0 : (rows <= 32 ? 1 : 2), lkg = 2 - lrt, lsg = (S == 16 ? 4 : 3) - lkg;
    static_assert(kManyWarps == 4 && (S == 8 || S == 16), "powers of two above");
    const int RT = 1 << lrt, KG = 1 << lkg, SG = 1 << lsg;
    const int first_row = (int)(blockIdx.x >> lr) * 16 * RT, row_step = (int)(gridDim.x >> lr) * 16 * RT;
    if (first_row >= rows) return;
    if (tid < S) {
        mbar_init(&full[tid], TMA ? 1 : 32);
        mbar_init(&empty[tid], RT);
    }
    fence_mbar_init();
    __syncthreads();
    const int tiles = (r.keys + kTile - 1) / kTile;
    const int first = (tiles * rank) >> lr, mine = ((tiles * (rank + 1)) >> lr) - first;
    cg::cluster_group cl = cg::this_cluster();
    SlabWait slab_wait;
    // keys few enough that K and V fill the ring once and stay, for the only block of
    // rows there is: K tile i in slot i, V tile i in slot S/2 + i. (Not at 128 channels,
    // where the ring would hold 256 keys and the registers are needed elsewhere.)
    const bool resident = D == 64 && mine <= S / 2 && first_row + row_step >= rows;

    if (warp == kManyWarps) {  // the feeder: K tiles, then K and V tiles in turn, for every block of rows
        const int8_t *kbase = a.k + kvh * a.head_stride, *vbase = a.v + kvh * a.head_stride;
        // lane i holds the page of box i of a window of 32 boxes (the table's latency
        // would otherwise be paid for every slot); boxes of at most 32 rows
        const int box = min(1 << a.page_log2, 32), per = 32 / box;
        int32_t pages = -1;
        auto window = [&](int i) {
            const int j = first * kTile + i * 32 + lane * box;
            pages = j < min((first + mine) * kTile, r.keys) ? r.table[j >> a.page_log2] : -1;
            if ((uint32_t)pages >= a.n_pages) pages = -1;
        };
        if (TMA) window(0);
        // a slot filled from half tile i (32 keys): with its K and the next's, its V and
        // the next's, or its K and its V
        enum { kKeys, kValues, kBoth };
        auto fill = [&](uint32_t slot, int i, int what) {
            uint8_t *dst = smem + slot * F::kBytes;
            const int j0 = first * kTile + i * 32;
            if (TMA) {
                const int w = (i * per) & 31;
                if (w == 0 && mine * 2 * per > 32) window(i);
                const int32_t page = __shfl_sync(0xffffffffu, pages, what == kBoth ? w + (lane & (per - 1)) : w + lane);
                const bool ok = lane < 2 * per && page >= 0;
                const uint32_t n_box = __popc(__ballot_sync(0xffffffffu, ok));
                if (lane == 0) mbar_arrive_expect_tx(&full[slot], n_box * box * D);
                __syncwarp();
                const bool v = what == kValues || (what == kBoth && lane >= per);
                const int j = j0 + (what == kBoth && v ? lane - per : lane) * box;
                if (ok)
                    tma_load_4d(v ? &tmap_v : &tmap_k, &full[slot], dst + lane * box * D, 0, j & ((1 << a.page_log2) - 1), kvh,
                                page);
            } else {
                load_rows<D, 32 * D>(a, r, what == kValues ? vbase : kbase, j0, dst);
                load_rows<D, 32 * D>(a, r, what == kKeys ? kbase : vbase, what == kBoth ? j0 : j0 + 32, dst + 32 * D);
                mbar_arrive_cp_async(&full[slot]);
            }
        };
        if (resident) {
            for (int i = 0; i < mine; ++i) fill(i, 2 * i, kKeys);
            for (int i = 0; i < mine; ++i) fill(S / 2 + i, 2 * i, kValues);
            if (ranks > 1) cl.sync(), cl.sync(), cl.sync();
            __syncthreads();
            return;
        }
        uint32_t done = 0;  // blocks of rows fed
        // place `at` of a set's slots in this block of rows
        auto put = [&](int set, int at, int i, bool pass2) {
            const uint32_t count = (mine - set + KG - 1) >> lkg, n = 3 * count * done + (pass2 ? count : 0) + at;
            const uint32_t slot = (set << lsg) + (n & (SG - 1));
            if (n >= SG) slab_wait(&empty[slot], ((n >> lsg) - 1) & 1);
            fill(slot, i, pass2 ? kBoth : kKeys);
        };
        auto put2 = [&](int i) {  // half tile i of the second pass
            const int tile = i >> 1;
            put(tile & (KG - 1), 2 * (tile >> lkg) + (i & 1), i, true);
        };
        for (int row0 = first_row; row0 < rows; row0 += row_step, ++done) {
            for (int i = 0; i < mine; ++i) put(i & (KG - 1), i >> lkg, 2 * i, false);
            // a ring of the second pass's slots goes out before the blocks meet
            const int ahead = min(S, 2 * mine);
            for (int i = 0; i < ahead; ++i) put2(i);
            if (ranks > 1) cl.sync();
            for (int i = ahead; i < 2 * mine; ++i) put2(i);
            if (ranks > 1) cl.sync(), cl.sync();
            __syncthreads();  // the ring is free of sums
        }
        return;
    }

    const int rt = warp & (RT - 1), kg = warp >> lrt;
    const RrsK rk = rrs_k(a.qk_shift);
    const FastExp fx = fast_exp(a);
    const FinishK fk{rrs_k(a.rsqrt_offset), rrs_k(a.av_shift), a.av_mult};
    const bool fast_ok = a.frac_bits >= 7 && a.frac_bits <= 14 && a.qk_shift >= 1 && a.qk_shift <= 9;
    const int cut = min(22795, 8 << min(max(a.frac_bits, 7), 14));
    auto requant = [&](int32_t acc) { return clampi(rrs_apply(wmul(acc, a.qk_mult), rk), -32768, 32767); };
    auto meet = [&] {
        if (ranks > 1) cl.sync();
        else asm volatile("bar.sync 1, %0;" ::"n"(32 * kManyWarps) : "memory");
    };
    // the key, of 16, whose row a lane loads for column n = 2t'+e of score tile jj:
    // operand byte 4t' + 2jj + e of P is that of key order(4t' + 2jj + e). 128-byte
    // rows need another order than 64-byte ones so that neither the K nor the V
    // fragments meet bank conflicts
    auto order = [](int k) { return D == 64 ? k : 8 * (k >> 3) + 4 * (k & 1) + 2 * ((k >> 1) & 1) + ((k >> 2) & 1); };
    // lane offsets in a tile: its K piece of score tile jj and 64-byte half h, its V
    // row of piece 0 (piece c: the same with bits 4.. flipped by c)
    uint32_t koff[2][D / 64];
#pragma unroll
    for (int jj = 0; jj < 2; ++jj)
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
            const int row = order(4 * (g >> 1) + 2 * jj + (g & 1));
            koff[jj][h] = row * D + swz<D>(row, 4 * h + t) * 16;
        }
    const int vrow = (lane & 16) + order(lane & 15);
    const uint32_t voff = vrow * D + swz<D>(vrow, 0) * 16;

    bool holes = false;  // keys of this block without a page
    for (int j = (((first * kTile) >> a.page_log2) + lane) << a.page_log2; j < min((first + mine) * kTile, r.keys);
         j += 32 << a.page_log2)
        holes |= !has_page(a, r, j);
    const int all_see = __any_sync(0xffffffffu, holes) ? 0 : min(r.ctx, r.keys);  // keys below are seen by every row

    uint32_t n = 0;  // tiles of this set's slots seen so far
    auto slot = [&](uint32_t n) { return (kg << lsg) + (n & (SG - 1)); };
    const uint32_t ring = smem_u32(smem);
    auto tile_at = [&](uint32_t n) { return ring + slot(n) * F::kBytes; };
    auto arrived = [&](uint32_t n) { slab_wait(&full[slot(n)], (n >> lsg) & 1); };
    auto release = [&](uint32_t n) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[slot(n)]);
    };
    for (int row0 = first_row; row0 < rows; row0 += row_step) {
        const int ra = row0 + 16 * rt + g, rb = ra + 8;  // this lane's rows
        const int ta = G == 1 ? ra : ra / G, tb = G == 1 ? rb : rb / G;
        // the 16-row operand of step s of half c: bytes 16t + 8s.. and 16t + 8s + 4.. of
        // rows ra, rb. Loaded word by word: out of 16-byte loads the compiler moved the
        // registers into operand order again for every product
        uint32_t q[D / 64][2][4];
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                auto word = [&](int row, int tok) -> uint32_t {
                    if (row >= rows) return 0;
                    return *reinterpret_cast<const uint32_t *>(a.q + (int64_t)(r.first + tok) * a.ldq +
                                                               (int64_t)(kvh * G + row - tok * G) * a.q_hs + 64 * c + 16 * t + 4 * x);
                };
                q[c][x >> 1][2 * (x & 1)] = word(ra, ta);
                q[c][x >> 1][2 * (x & 1) + 1] = word(rb, tb);
            }
        if (tid < 64) s_sum[tid] = 0, s_max[tid] = INT32_MIN;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kManyWarps) : "memory");

        // which keys j0 .. j0+31 the rows ra and rb see; true when all of them by all
        auto seen = [&](int j0, uint32_t &wa, uint32_t &wb) {
            if (j0 + 32 <= all_see) return true;
            wa = wb = __ballot_sync(0xffffffffu, has_page(a, r, j0 + lane));
            if (j0 + 32 <= r.ctx) return false;
            const int u0 = j0 - r.ctx;  // place of the first key among the new tokens
            auto word = [&](int n) -> uint32_t {
                if (a.words == 0) return n < u0 ? 0u : (n - u0 >= 31 ? 0xffffffffu : (2u << (n - u0)) - 1);
                if (n >= r.fresh) return 0;
                const int32_t *m = a.mask + (int64_t)(r.first + n) * a.words;
                auto at = [&](int w) -> uint32_t { return w < 0 ? 0xffffffffu : (w < a.words ? (uint32_t)m[w] : 0u); };
                return __funnelshift_r(at(u0 >> 5), at((u0 >> 5) + 1), u0 & 31);
            };
            wa &= word(ta);
            wb &= word(tb);
            return false;
        };
        // raw scores of 32 keys: c[2 * half + jj], columns order(4t + 2jj + e) + 16 * half
        auto raw = [&](int32_t (&c)[4][4], uint32_t ks) {
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
                int4 k[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) k[j] = lds_v4(ks + 16 * (j >> 1) * D + koff[j & 1][h]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t (&w)[4] = q[h][0];
                    if (h == 0) mma_s8_first(c[j], w[0], w[1], w[2], w[3], k[j].x, k[j].y);
                    else mma_s8(c[j], w[0], w[1], w[2], w[3], k[j].x, k[j].y);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) mma_s8(c[j], q[h][1][0], q[h][1][1], q[h][1][2], q[h][1][3], k[j].z, k[j].w);
            }
        };
        auto bit = [&](int j, int e) { return 16 * (j >> 1) + order(4 * t + 2 * (j & 1) + e); };

        int32_t m0 = INT32_MIN, m1 = INT32_MIN;
        auto tile_max = [&](auto masked, int i) {
            if (resident) slab_wait(&full[i], 0);
            else arrived(n);
            const uint32_t ks = resident ? ring + i * F::kBytes : tile_at(n);
#pragma unroll
            for (int h32 = 0; h32 < 2; ++h32) {
                int32_t c[4][4];
                raw(c, ks + h32 * 32 * D);
                uint32_t wa, wb;
                if (masked && !seen((first + i) * kTile + 32 * h32, wa, wb)) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            if (!((wa >> bit(j, e)) & 1)) c[j][e] = INT32_MIN;
                            if (!((wb >> bit(j, e)) & 1)) c[j][2 + e] = INT32_MIN;
                        }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    m0 = max(m0, max(c[j][0], c[j][1]));
                    m1 = max(m1, max(c[j][2], c[j][3]));
                }
            }
            if (!resident) release(n);
        };
        // tiles that every row sees whole have loops of their own: the code for the
        // others beside it cost the hot loop a sixth of its speed
        int i1 = kg;
        for (; i1 < mine && (first + i1 + 1) * kTile <= all_see; i1 += KG, ++n) tile_max(std::false_type(), i1);
        for (; i1 < mine; i1 += KG, ++n) tile_max(std::true_type(), i1);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            m0 = max(m0, __shfl_xor_sync(0xffffffffu, m0, o));
            m1 = max(m1, __shfl_xor_sync(0xffffffffu, m1, o));
        }
        if (t == 0) atomicMax(&s_max[16 * rt + g], m0), atomicMax(&s_max[16 * rt + g + 8], m1);
        meet();
        if (ranks == 1) {
            m0 = s_max[16 * rt + g];
            m1 = s_max[16 * rt + g + 8];
        } else {
            m0 = cluster_max(cl, s_max + 16 * rt + g, ranks);
            m1 = cluster_max(cl, s_max + 16 * rt + g + 8, ranks);
        }
        const int32_t xa = (m0 == INT32_MIN ? -32768 : requant(m0)) + 1, xb = (m1 == INT32_MIN ? -32768 : requant(m1)) + 1;
        auto inside = [&](int32_t xm) { return xm <= 32767 && xm - cut > -32768; };
        const int64_t base_a = fast_base(xa, fx), base_b = fast_base(xb, fx);
        const bool fast = __all_sync(0xffffffffu, fast_ok && (ra >= rows || inside(xa)) && (rb >= rows || inside(xb)));

        // (P.V)^T: channels 16i + g (and + 8) of rows 2t, 2t+1 of either 8 rows
        int32_t o[D / 16][2][4];
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) o[i][e >> 2][e & 3] = 0;
        uint32_t sum0 = 0, sum1 = 0;
        auto key0 = [&](int i) { return (first + kg + (i >> 1) * KG) * kTile + 32 * (i & 1); };
        // half tile i of this set; hot: seen whole by rows that take the short exponential
        auto half_tile = [&](auto hot, int i) {
            const int tile = kg + (i >> 1) * KG, j0 = key0(i);
            uint32_t p[4];
            if (!resident) arrived(n);
            const uint32_t half = 32 * (i & 1) * D;
            const uint32_t ks = resident ? ring + tile * F::kBytes + half : tile_at(n);
            const uint32_t vs = voff + (resident ? ring + (S / 2 + tile) * F::kBytes + half : ks + 32 * D);
            {
                int32_t c[4][4];
                raw(c, ks);
                if (hot || fast) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[j][e] = (int32_t)fast_prob<false>(c[j][e], e < 2 ? base_a : base_b, 0, fx);
                } else if (fast_ok) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            c[j][e] = (int32_t)fast_prob<true>(c[j][e], e < 2 ? base_a : base_b,
                                                               kBias - 32768 - (e < 2 ? xa : xb), fx);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            c[j][e] = shift_exp_one(requant(c[j][e]), (int16_t)(e < 2 ? xa : xb), a.frac_bits);
                }
                auto pack = [](int32_t x, int32_t y, int32_t z, int32_t w) {
                    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
                };
                p[0] = pack(c[0][0], c[0][1], c[1][0], c[1][1]);
                p[1] = pack(c[0][2], c[0][3], c[1][2], c[1][3]);
                p[2] = pack(c[2][0], c[2][1], c[3][0], c[3][1]);
                p[3] = pack(c[2][2], c[2][3], c[3][2], c[3][3]);
            }
            uint32_t wa, wb;
            if (!hot && !seen(j0, wa, wb)) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t w = (x & 1) ? wb : wa;
                    uint32_t keep = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if ((w >> (16 * (x >> 1) + order(4 * t + e))) & 1) keep |= 0xffu << (8 * e);
                    p[x] &= keep;
                }
            }
            sum0 = __dp4a(p[0], 0x01010101u, __dp4a(p[2], 0x01010101u, sum0));
            sum1 = __dp4a(p[1], 0x01010101u, __dp4a(p[3], 0x01010101u, sum1));
            if (resident) slab_wait(&full[S / 2 + tile], 0);
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                uint32_t v[4];
                ldsm_trans_b8(v, vs ^ (16 * c));
                mma_s8u8(o[c][0], v[0], v[1], v[2], v[3], p[0], p[2]);
                mma_s8u8(o[c][1], v[0], v[1], v[2], v[3], p[1], p[3]);
            }
            if (!resident) release(n);
        };
        const int halves = 2 * ((mine - kg + KG - 1) >> lkg);
        int i2 = 0;
        if (fast)
            for (; i2 < halves && key0(i2) + 32 <= all_see; ++i2, ++n) half_tile(std::true_type(), i2);
        for (; i2 < halves; ++i2, ++n) half_tile(std::false_type(), i2);
        // sums over the warps that shared the tiles, then over the cluster
        sum0 += __shfl_xor_sync(0xffffffffu, sum0, 1);
        sum1 += __shfl_xor_sync(0xffffffffu, sum1, 1);
        sum0 += __shfl_xor_sync(0xffffffffu, sum0, 2);
        sum1 += __shfl_xor_sync(0xffffffffu, sum1, 2);
        auto give = [&](int32_t *d, int32_t v) {
            if (KG > 1) atomicAdd(d, v);
            else *d = v;
        };
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kManyWarps) : "memory");  // every tile has been read
        if (KG > 1) {
            for (int i = tid; i < 16 * RT * OLD / 4; i += 32 * kManyWarps)
                reinterpret_cast<int4 *>(s_o)[i] = make_int4(0, 0, 0, 0);
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kManyWarps) : "memory");
        }
        if (t == 0) give(&s_sum[16 * rt + g], (int32_t)sum0), give(&s_sum[16 * rt + g + 8], (int32_t)sum1);
        int32_t *d0 = s_o + (16 * rt + 2 * t) * OLD + g;
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                int32_t *d = d0 + 8 * e * OLD + 16 * c;
                give(d, o[c][e][0]), give(d + OLD, o[c][e][1]), give(d + 8, o[c][e][2]), give(d + OLD + 8, o[c][e][3]);
            }
        meet();
        // rows dealt out over the cluster and the warps, four channels per lane
        constexpr int kAtOnce = 128 / D;  // rows per step of a warp
        const int nr = min(16 * RT, rows - row0), first_k = (rank * kManyWarps + warp) * kAtOnce, step = ranks * kManyWarps * kAtOnce;
        int32_t inv = 0;  // of the warp's row first_k + (lane / kAtOnce) * step + lane % kAtOnce
        {
            const int k = first_k + lane / kAtOnce * step + lane % kAtOnce;
            if (k < nr) inv = fisr(ranks == 1 ? s_sum[k] : cluster_sum(cl, s_sum + k, ranks), a.rsqrt_offset);
        }
#pragma unroll 1
        for (int k0 = first_k, i = 0; k0 < nr; k0 += step, i += kAtOnce) {
            const int k = k0 + lane / (D / 4), d = lane % (D / 4) * 4, row = row0 + k, tok = G == 1 ? row : row / G;
            const int32_t v = __shfl_sync(0xffffffffu, inv, i + lane / (D / 4));
            if (k < nr) {
                int32_t *p = s_o + k * OLD + d;
                const int4 x = ranks == 1 ? *reinterpret_cast<const int4 *>(p) : cluster_sum4(cl, p, ranks);
                *reinterpret_cast<uint32_t *>(a.y + (int64_t)(r.first + tok) * a.ldy + (int64_t)(kvh * G + row - tok * G) * D +
                                              d) = finish4(fk, x, v);
            }
        }
        meet();  // no block's sums go away or are cleared while another reads them
        fence_proxy_async_smem();
        __syncthreads();  // the feeder may fill the ring again
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
static cudaError_t cache_maps(const TreeAttnArgs &a, int box_rows, CacheMaps &m) {
    const uint64_t sizes[4] = {(uint64_t)a.D, 1ull << a.page_log2, (uint64_t)a.Hkv, a.n_pages};
    const uint64_t strides[3] = {a.row_stride, (uint64_t)a.head_stride, a.page_stride};
    const uint32_t box[4] = {(uint32_t)a.D, std::min(1u << a.page_log2, (unsigned)box_rows), 1, 1};
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
    // A request of many rows among others of few takes 8 at a time; a batch of single
    // tokens has no such request. Fewer at a time too while the SMs have fewer than 4
    // warps each: a warp's time goes by its rows (7 rows of 12 keys on 6 heads: 16 us
    // by one warp a head, 10 by one a row)
    const int64_t guess = std::min<int64_t>(kFewRows, mean_rows);
    if (a.N <= a.B)
        while (p.group >= 2 * guess) p.group /= 2;
    while (p.group > 1 && pairs * p.warps * p.ranks * ((guess + p.group - 1) / p.group) < 4 * num_sms()) p.group /= 2;
    p.row_blocks = (int)((guess + p.group - 1) / p.group);
    // room for the scores of every slab
    const int64_t per_warp = (keys / Slab<D>::kKeys / p.ranks + p.warps) / p.warps;
    p.slots = (int)std::min<int64_t>(64, std::max<int64_t>(p.group, per_warp * std::min<int64_t>(p.group, guess)));
    return p.group == 1 ? few_rows_warps<D, 1>(a, m, tma, p, st) : few_rows_warps<D, kFewRows>(a, m, tma, p, st);
}

template <int D, bool TMA>
static cudaError_t many_rows(const TreeAttnArgs &a, const CacheMaps &m, int64_t mean_rows, cudaStream_t st) {
    const int64_t keys = std::max<int64_t>(1, (int64_t)a.width << a.page_log2), pairs = (int64_t)a.B * a.Hkv;
    // a row block per 64 rows: as many as the tree mask allows, at most twice the mean's
    const int64_t most = (a.words ? std::min<int64_t>(a.N, 32 * a.words) : a.N) * a.G;
    const int row_blocks = (int)std::min<int64_t>(1024, (std::min(most, 2 * mean_rows) + 63) / 64);
    // split the keys while there are fewer than four blocks per SM and a block
    // keeps 256 keys
    int ranks = 1;
    while (ranks < 8 && pairs * row_blocks * ranks < 4 * num_sms() && keys / ranks > 256) ranks *= 2;
    const size_t smem = Many<D>::smem();
    static SmemLimit lim;
    cudaError_t e = raise_smem_limit(many_rows_kernel<D, TMA>, smem, lim);
    if (e != cudaSuccess) return e;
    return launch_cluster(many_rows_kernel<D, TMA>, ranks, dim3(ranks * row_blocks, a.Hkv, a.B), dim3(32 * (kManyWarps + 1)), smem, st,
                          m.k, m.v, a, ranks);
}

template <int D>
static cudaError_t attention(const TreeAttnArgs &a, cudaStream_t st) {
    // tensor maps need pages of 8 rows or more and axes that step
    const bool tma = a.page_log2 >= 3 && a.n_pages > 0 && a.row_stride > 0 && a.head_stride > 0 && a.page_stride > 0;
    // the batch's mean decides for all of it; either kernel takes any count
    const int64_t mean_rows = (a.N + a.B - 1) / a.B * a.G;
    const bool many = mean_rows > kFewRows;
    CacheMaps m = {};
    if (tma)
        if (cudaError_t e = cache_maps(a, many ? 32 : Slab<D>::kKeys, m); e != cudaSuccess) return e;
    if (!many) return few_rows<D>(a, m, tma, mean_rows, st);
    return tma ? many_rows<D, true>(a, m, mean_rows, st) : many_rows<D, false>(a, m, mean_rows, st);
}

}  // namespace tree

cudaError_t tree_attention(const TreeAttnArgs &a, cudaStream_t st) {
    if (a.B == 0) return cudaMemset2DAsync(a.y, a.ldy, 0, (size_t)a.H * a.D, (size_t)a.N, st);
    TreeAttnArgs b = a;
    b.largest_first = a.B > 1 && a.B <= 32 && ((int64_t)a.width << a.page_log2) > 1024;
    return a.D == 64 ? tree::attention<64>(b, st) : tree::attention<128>(b, st);
}

}  // namespace iw
