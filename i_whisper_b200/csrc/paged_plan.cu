// paged_plan.cu -- one decoding step's plan (block tables, slot map,
// positions, ancestor masks) from request lengths, and the write of new K/V
// rows into the pages of the INT8 cache.
#include "iw_common.cuh"
#include "paged.cuh"

namespace iw {

// ---------------------------------------------------------------------------
// iw_paged_plan. Two prefix sums over the requests place everything:
//   starts_b = sum of new tokens before b      (rows of the step)
//   off_b    = sum of needed pages before b    (places in the free list)
// with have = ceil(ctx/P), want = min(ceil((ctx+new)/P), width) and
// need = max(0, want - have). Every block computes both sums for itself in
// shared memory, so that one launch does the whole plan, at 8*B bytes from L2 per
// block. Bound by latency (launch, lengths, scan, search): 8 requests of up to 7
// tokens 3.7 us, 1024 trees of 16 to 64 tokens 6.1 us.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 256;
constexpr int32_t kPlanMaxLen = 1 << 30;

IW_DEV int32_t plan_cap(int64_t v) { return (int32_t)(v < INT32_MAX ? v : INT32_MAX); }

struct PlanReq {
    int32_t ctx, fresh;
    int64_t have, want;  // pages
    int32_t need;
};

IW_DEV PlanReq plan_request(const PlanArgs &a, int b, int &bad) {
    PlanReq r;
    r.ctx = a.ctx[b];
    r.fresh = a.fresh[b];
    if (r.ctx < 0 || r.ctx > kPlanMaxLen) r.ctx = 0, bad |= 8;
    if (r.fresh < 0 || r.fresh > kPlanMaxLen) r.fresh = 0, bad |= 8;
    const int64_t p1 = ((int64_t)1 << a.page_log2) - 1;
    r.have = (r.ctx + p1) >> a.page_log2;
    r.want = ((int64_t)r.ctx + r.fresh + p1) >> a.page_log2;
    if (r.want > a.width) bad |= 2;
    const int64_t n = (r.want < a.width ? r.want : (int64_t)a.width) - r.have;
    r.need = n > 0 ? (int32_t)n : 0;
    if (a.words && r.fresh > a.max_new) bad |= 16;
    return r;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PlanArgs a) {
    pdl_wait();
    pdl_launch();
    // starts [B + 1], then off [B + 1]. The sums run in 64 bits and are kept
    // capped at 2^31 - 1: no row or free page has an index that large, so
    // what a capped sum places is past the end either way.
    extern __shared__ int32_t plan_sums[];
    int32_t *s_start = plan_sums, *s_off = plan_sums + a.B + 1;
    __shared__ int64_t w_tok[kPlanThreads / 32], w_pg[kPlanThreads / 32];
    __shared__ int s_bad;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    // each thread sums a run of consecutive requests
    const int run = (a.B + kPlanThreads - 1) / kPlanThreads;
    const int b0 = min(tid * run, a.B), b1 = min(b0 + run, a.B);
    int64_t tok = 0, pg = 0;
    int bad = 0;
    for (int b = b0; b < b1; ++b) {
        const PlanReq r = plan_request(a, b, bad);
        tok += r.fresh;
        pg += r.need;
    }
    if (bad) atomicOr(&s_bad, bad);
    int64_t tok_i = tok, pg_i = pg;  // inclusive scans
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t t = __shfl_up_sync(0xffffffffu, tok_i, o), p = __shfl_up_sync(0xffffffffu, pg_i, o);
        if (lane >= o) tok_i += t, pg_i += p;
    }
    if (lane == 31) w_tok[warp] = tok_i, w_pg[warp] = pg_i;
    __syncthreads();
    tok = tok_i - tok;
    pg = pg_i - pg;
    for (int w = 0; w < warp; ++w) tok += w_tok[w], pg += w_pg[w];
    for (int b = b0; b < b1; ++b) {
        s_start[b] = plan_cap(tok);
        s_off[b] = plan_cap(pg);
        int ignored = 0;
        const PlanReq r = plan_request(a, b, ignored);
        tok += r.fresh;
        pg += r.need;
    }
    if (b1 == a.B && (b0 < b1 || tid == kPlanThreads - 1)) s_start[a.B] = plan_cap(tok), s_off[a.B] = plan_cap(pg);
    __syncthreads();

    const int64_t total = s_start[a.B], pages = s_off[a.B];
    int64_t head = *a.free_head;
    head = head < 0 ? 0 : (head > a.n_free ? a.n_free : head);
    auto granted = [&](int64_t at) -> int32_t { return head + at < a.n_free ? a.free_pages[head + at] : -1; };
    const int64_t gtid = (int64_t)blockIdx.x * kPlanThreads + tid, gsize = (int64_t)gridDim.x * kPlanThreads;
    for (int64_t b = gtid; b <= a.B; b += gsize) a.starts[b] = s_start[b];
    // table entries: one warp per request
    for (int64_t b = gtid >> 5; b < a.B; b += gsize >> 5) {
        int ignored = 0;
        const PlanReq r = plan_request(a, (int)b, ignored);
        for (int64_t j = lane; j < r.need; j += 32) a.table[b * a.table_ld + r.have + j] = granted((int64_t)s_off[b] + j);
    }
    // tokens
    for (int64_t i = gtid; i < a.max_tokens; i += gsize) {
        int64_t slot = -1;
        int32_t req = -1, pos = 0;
        int32_t *mrow = a.words ? a.mask + i * a.words : nullptr;
        for (int w = 0; w < a.words; ++w) mrow[w] = 0;
        if (i < total) {
            int lo = 0, hi = a.B - 1;  // last b with starts[b] <= i; requests without new tokens never are
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s_start[mid] <= i) lo = mid;
                else hi = mid - 1;
            }
            req = lo;
            int ignored = 0;
            const PlanReq r = plan_request(a, req, ignored);
            const int64_t t = i - s_start[req];
            const int64_t place = r.ctx + t, col = place >> a.page_log2;
            int32_t page = -1;
            if (col < a.width)
                page = col < r.have ? a.table[(int64_t)req * a.table_ld + col] : granted(s_off[req] + (col - r.have));
            if (page >= 0) slot = ((int64_t)page << a.page_log2) + (place & (((int64_t)1 << a.page_log2) - 1));
            if (a.parents) {
                // walk to the root; indices fall strictly, so the walk ends
                int64_t depth = 0;
                for (int64_t u = t; u >= 0;) {
                    if ((u >> 5) < a.words) mrow[u >> 5] |= (int32_t)(1u << (u & 31));
                    const int64_t p = a.parents[(int64_t)s_start[req] + u];
                    if (p < 0 || p >= u) break;
                    u = p;
                    ++depth;
                }
                pos = (int32_t)(r.ctx + depth);
            } else {
                pos = (int32_t)place;
            }
        }
        a.slots[i] = slot;
        a.request[i] = req;
        a.position[i] = pos;
    }
    if (blockIdx.x == 0 && tid == 0) {
        *a.status = s_bad | (head + pages > a.n_free ? 1 : 0) | (total > a.max_tokens ? 4 : 0);
        *a.free_head_out = (int32_t)min(head + pages, a.n_free);
    }
}

cudaError_t paged_plan(const PlanArgs &a, cudaStream_t st) {
    const int64_t rows = a.max_tokens > a.B + 1 ? a.max_tokens : a.B + 1;
    int64_t blocks = (rows + kPlanThreads - 1) / kPlanThreads;
    if (blocks > 2 * num_sms()) blocks = 2 * num_sms();
    const size_t smem = 2 * (size_t)(a.B + 1) * sizeof(int32_t);
    static SmemLimit lim;
    cudaError_t e = raise_smem_limit(paged_plan_kernel, smem, lim);
    if (e != cudaSuccess) return e;
    return launch_pdl(paged_plan_kernel, dim3((unsigned)blocks), dim3(kPlanThreads), smem, st, a);
}

// ---------------------------------------------------------------------------
// iw_paged_kv_write. A copy: each thread 16 bytes of K and of V, a token's row of
// one head (64 or more bytes) read and written whole. Bound by latency at one
// step's tokens (256 tokens, 16 heads of 64: 1.6 us) and by HBM at many: 40001
// tokens of 20 heads of 64 to slots in random order 44 us, 4.7 TB/s of reads
// and 64-byte writes; 2, 4 or 8 pieces per thread in flight measured 44, 44 and
// 50 us, and 1.8, 2.8 and 5.3 us for the step.
// ---------------------------------------------------------------------------
constexpr int kWriteThreads = 256;
__global__ void __launch_bounds__(kWriteThreads) paged_kv_write_kernel(KvWriteArgs a, uint32_t per, uint32_t pieces) {
    pdl_wait();
    pdl_launch();
    const int64_t total = a.N * per, i = (int64_t)blockIdx.x * kWriteThreads + threadIdx.x;
    if (i >= total) return;
    const int64_t n = total <= UINT32_MAX ? (int64_t)((uint32_t)i / per) : i / per;
    const uint32_t r = (uint32_t)(i - n * per), h = r / pieces, c = (r - h * pieces) * 16;
    const int64_t slot = a.slots[n];
    if (slot < 0 || slot >= a.n_slots) return;
    const int64_t at = (slot >> a.page_log2) * a.page_stride + h * a.head_stride +
                       (slot & (((int64_t)1 << a.page_log2) - 1)) * a.row_stride + c;
    const int4 kk = *reinterpret_cast<const int4 *>(a.k + n * a.ldk + h * a.k_hs + c);
    const int4 vv = *reinterpret_cast<const int4 *>(a.v + n * a.ldv + h * a.v_hs + c);
    *reinterpret_cast<int4 *>(a.k_cache + at) = kk;
    *reinterpret_cast<int4 *>(a.v_cache + at) = vv;
}

cudaError_t paged_kv_write(const KvWriteArgs &a, cudaStream_t st) {
    const uint32_t pieces = (uint32_t)(a.D >> 4), per = pieces * (uint32_t)a.H;
    const int64_t blocks = (a.N * per + kWriteThreads - 1) / kWriteThreads;
    if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
    return launch_pdl(paged_kv_write_kernel, dim3((unsigned)blocks), dim3(kWriteThreads), 0, st, a, per, pieces);
}

}  // namespace iw
