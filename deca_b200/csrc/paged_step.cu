// The bookkeeping of one serving step on the device (deca_paged_step): token and page prefix sums
// over the requests, pages from the free list into the block tables, a position and a cache slot for
// every token.
//
// The work is a few bytes per token; what counts is that it is one launch without a hand-over between
// CTAs.  Every CTA therefore repeats the prefix sums over all requests (8 bytes a request, from L2)
// in its own shared memory and then takes its share of the tokens and of the new pages.  A page that
// the step hands out is computed from its rank in the free list by whoever needs it and never read back
// from the table, so the CTAs are independent of each other.
//
// Bound by latency: 8 requests 3.0 - 3.3 us, 512 requests with 76 800 token rows 4.8 - 5.1 us (CTAs of 1024 threads, whose
// warp sums one thread after the other adds up, took 7.0 and 8.7).
#include "common.cuh"
#include "ptx.cuh"

namespace deca {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRequests = 8192;

struct StepArgs {
    const int *ctx, *add;
    int *table;
    long long table_stride;
    const int *free_pages, *n_free;
    int B, W, free_cap;
    int page_shift;
    long long T;
    int *cu, *kv, *pos;
    long long *slots;
    int *n_free_out, *short_out;
};

struct Request {
    int ctx, add;  // cached tokens, new tokens
    int held;      // table entries in use before the step
    int need;      // entries the step adds
    int kv;        // cached tokens after the step
};

__device__ __forceinline__ Request request_of(const StepArgs &g, int r) {
    Request q;
    q.ctx = max(g.ctx[r], 0);
    q.add = max(g.add[r], 0);
    const long long room = (long long)g.W << g.page_shift;
    const long long kv = min((long long)q.ctx + q.add, room), page = 1ll << g.page_shift;
    q.kv = (int)min(kv, 2147483647ll);
    q.held = (int)min((q.ctx + page - 1) >> g.page_shift, (long long)g.W);
    q.need = max((int)((q.kv + page - 1) >> g.page_shift) - q.held, 0);
    return q;
}

// Sums of lengths stop at the largest int: a prefix then never turns negative, whatever the lengths are.
__device__ __forceinline__ int sat_add(int a, int b) { return (int)min((long long)a + b, 2147483647ll); }

// largest r with prefix[r] <= x among 0 .. n - 1
__device__ __forceinline__ int find(const int *prefix, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] <= x)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kThreads) paged_step_kernel(const StepArgs g) {
    extern __shared__ int smem[];
    int *tok = smem;                // [B] first token of each request
    int *pages = smem + g.B;        // [B] first of its new pages in the order of the step
    int *ctx_of = smem + 2 * g.B;   // [B]
    __shared__ int warp_tok[kWarps], warp_pages[kWarps];
    const int free_given = *g.n_free;  // on its way while the lengths are summed
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (g.B + kThreads - 1) / kThreads;
    const int r0 = min(tid * per, g.B), r1 = min(r0 + per, g.B);

    int my_tok = 0, my_pages = 0;
    for (int r = r0; r < r1; ++r) {
        const Request q = request_of(g, r);
        tok[r] = my_tok;
        pages[r] = my_pages;
        ctx_of[r] = q.ctx;
        my_tok = sat_add(my_tok, q.add);
        my_pages = sat_add(my_pages, q.need);
    }
    int inc_tok = my_tok, inc_pages = my_pages;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int a = __shfl_up_sync(0xFFFFFFFFu, inc_tok, s), b = __shfl_up_sync(0xFFFFFFFFu, inc_pages, s);
        if (lane >= s) inc_tok = sat_add(inc_tok, a), inc_pages = sat_add(inc_pages, b);
    }
    if (lane == 31) warp_tok[warp] = inc_tok, warp_pages[warp] = inc_pages;
    // what the lanes before this one hold
    int base_tok = __shfl_up_sync(0xFFFFFFFFu, inc_tok, 1), base_pages = __shfl_up_sync(0xFFFFFFFFu, inc_pages, 1);
    if (lane == 0) base_tok = base_pages = 0;
    __syncthreads();
    // the warps' sums, scanned by every warp for itself
    int wt = lane < kWarps ? warp_tok[lane] : 0, wp = lane < kWarps ? warp_pages[lane] : 0;
#pragma unroll
    for (int s = 1; s < kWarps; s <<= 1) {
        const int a = __shfl_up_sync(0xFFFFFFFFu, wt, s), b = __shfl_up_sync(0xFFFFFFFFu, wp, s);
        if (lane >= s) wt = sat_add(wt, a), wp = sat_add(wp, b);
    }
    const int total_tok = __shfl_sync(0xFFFFFFFFu, wt, kWarps - 1), total_pages = __shfl_sync(0xFFFFFFFFu, wp, kWarps - 1);
    const int prev_tok = __shfl_sync(0xFFFFFFFFu, wt, max(warp - 1, 0)), prev_pages = __shfl_sync(0xFFFFFFFFu, wp, max(warp - 1, 0));
    if (warp > 0) base_tok = sat_add(base_tok, prev_tok), base_pages = sat_add(base_pages, prev_pages);
    for (int r = r0; r < r1; ++r) tok[r] = sat_add(tok[r], base_tok), pages[r] = sat_add(pages[r], base_pages);
    __syncthreads();

    const int n_free = min(max(free_given, 0), g.free_cap);
    auto held_of = [&](int ctx) {
        return (int)min(((long long)ctx + (1 << g.page_shift) - 1) >> g.page_shift, (long long)g.W);
    };
    auto fresh_page = [&](long long rank) { return rank < n_free ? g.free_pages[n_free - 1 - rank] : -1; };
    const long long first = (long long)blockIdx.x * kThreads + tid, step = (long long)gridDim.x * kThreads;

    for (long long t = first; t < g.T; t += step) {
        long long pos = 0, slot = -1;
        if (t < total_tok) {
            const int r = find(tok, g.B, (int)t);
            pos = (long long)ctx_of[r] + (t - tok[r]);
            if (pos >> g.page_shift < g.W) {
                const int e = (int)(pos >> g.page_shift), held = held_of(ctx_of[r]);
                const int page = e < held ? g.table[r * g.table_stride + e] : fresh_page((long long)pages[r] + e - held);
                if (page >= 0) slot = ((long long)page << g.page_shift) + (pos & ((1 << g.page_shift) - 1));
            }
        }
        g.pos[t] = (int)min(pos, 2147483647ll);
        g.slots[t] = slot;
    }
    for (long long i = first; i < total_pages; i += step) {
        const int r = find(pages, g.B, (int)i);
        g.table[r * g.table_stride + held_of(ctx_of[r]) + (i - pages[r])] = fresh_page(i);
    }
    for (long long r = first; r < g.B; r += step) {
        g.cu[r] = tok[r];
        g.kv[r] = request_of(g, (int)r).kv;
    }
    if (first == 0) {
        g.cu[g.B] = total_tok;
        *g.n_free_out = max(n_free - total_pages, 0);
        *g.short_out = max(total_pages - n_free, 0);
    }
}

}  // namespace
}  // namespace deca

using namespace deca;

extern "C" int deca_paged_step(const int32_t *ctx_lens, const int32_t *new_lens, int B, int32_t *block_table,
                               int64_t table_stride, int table_width, const int32_t *free_pages, int free_capacity,
                               const int32_t *n_free, int page_size, int64_t T, int32_t *cu_q, int32_t *kv_lens,
                               int32_t *positions, int64_t *slots, int32_t *n_free_out, int32_t *short_out, void *stream) {
    if (B < 1 || B > kMaxRequests || table_width < 1 || T < 0 || T > 2147483647ll || free_capacity < 0) return DECA_ERR_SHAPE;
    if (page_size < 1 || (page_size & (page_size - 1)) != 0 || page_size > (1 << 20)) return DECA_ERR_SHAPE;
    if ((int64_t)table_width * page_size > 2147483647ll) return DECA_ERR_SHAPE;
    if (table_stride < table_width) return DECA_ERR_SHAPE;
    if (!ctx_lens || !new_lens || !block_table || !n_free || !cu_q || !kv_lens || !n_free_out || !short_out) return DECA_ERR_NULL;
    if ((free_capacity > 0 && !free_pages) || (T > 0 && (!positions || !slots))) return DECA_ERR_NULL;
    // every CTA reads the inputs while others write
    struct Span {
        const void *at;
        int64_t bytes;
    };
    const Span in[] = {{ctx_lens, 4ll * B}, {new_lens, 4ll * B}, {free_pages, 4ll * free_capacity}, {n_free, 4},
                       {block_table, 4 * ((B - 1) * table_stride + table_width)}};
    const Span out[] = {{cu_q, 4ll * (B + 1)}, {kv_lens, 4ll * B}, {positions, 4 * T}, {slots, 8 * T}, {n_free_out, 4}, {short_out, 4}};
    auto meet = [](const Span &a, const Span &b) {
        const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
        return a.bytes > 0 && b.bytes > 0 && x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes;
    };
    for (int i = 0; i < 6; ++i) {
        for (const Span &s : in)
            if (meet(out[i], s)) return DECA_ERR_UNSUPPORTED;
        for (int j = 0; j < i; ++j)
            if (meet(out[i], out[j])) return DECA_ERR_UNSUPPORTED;
    }
    for (int i = 0; i < 4; ++i)
        if (meet(in[4], in[i])) return DECA_ERR_UNSUPPORTED;  // the table is written too
    for (const Span &sp : in)
        if (!aligned_to(sp.at, 4)) return DECA_ERR_ALIGN;
    for (const Span &sp : out)
        if (!aligned_to(sp.at, sp.at == slots ? 8 : 4)) return DECA_ERR_ALIGN;
    StepArgs g;
    g.ctx = ctx_lens, g.add = new_lens, g.table = block_table, g.table_stride = table_stride;
    g.free_pages = free_pages, g.n_free = n_free;
    g.B = B, g.W = table_width, g.free_cap = free_capacity;
    g.page_shift = 0;
    while ((1 << g.page_shift) < page_size) ++g.page_shift;
    g.T = T, g.cu = cu_q, g.kv = kv_lens, g.pos = positions;
    g.slots = reinterpret_cast<long long *>(slots);
    g.n_free_out = n_free_out, g.short_out = short_out;
    DeviceInfo di;
    if (int rc = current_device_info(&di)) return rc;
    const int64_t work = T > B ? T : B;
    int64_t grid = (work + kThreads - 1) / kThreads;
    if (grid > 4 * di.sms) grid = 4 * di.sms;
    static SmemLimitCache configured;
    const size_t smem = 3 * sizeof(int) * (size_t)B;
    if (int rc = ensure_dynamic_smem(paged_step_kernel, smem, configured)) return rc;
    paged_step_kernel<<<(unsigned)grid, kThreads, smem, static_cast<cudaStream_t>(stream)>>>(g);
    return (int)cudaGetLastError();
}
