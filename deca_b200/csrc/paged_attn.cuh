// What the two paged-attention schedules share: the device's view of the arguments, the list of work
// items, its division among the CTAs and the layout of partial results.
//
// Lengths live on the device, so the division is made there.  An item is one tile of query rows of one
// request and key head; row i of a tile packs token i / group and query head i % group of the key head, so
// all rows of an item read the same keys.  An item costs as many steps as it has key tiles (one at least: a
// row that sees no key is still written).  With U steps in all and G CTAs, CTA c takes the steps
// [U c / G, U (c + 1) / G) of the concatenated items: every CTA gets the same number of key tiles, whatever
// the lengths are.  An item that is cut leaves one partial result per CTA (fp32 numerators, maximum and
// sum per row), and a second kernel joins them in the order of the keys, so results do not depend on timing.
#pragma once

#include "ptx.cuh"

namespace deca {

struct PagedArgs {
    const char *q, *k, *v;
    char *o;
    long long q_st, q_sh, o_st, o_sh;                    // elements
    long long k_sp, k_sr, k_sh, v_sp, v_sr, v_sh;        // elements
    const int *table, *cu, *kv_lens;
    long long table_stride;
    long long T, num_pages;
    int B, W, Hkv, group;  // group: query heads per key head
    int page_shift;
    int causal;
    float sl2;  // scale * log2 e
    int whole;  // 1: items are not cut (no partial results)
    int min_steps;  // fewest steps worth a CTA of their own
    float *part;    // partial results, 2 per CTA
    struct PartialItem *meta;  // one per CTA
    DeviceStatus *status;
};

// The item that starts in a CTA's range and ends in a later one's; `last` < 0: none.
struct PartialItem {
    int req, head, tile, last;
};

struct ReqView {
    int q0, n;     // first row of Q, rows
    int kv;        // keys
    int shift;     // key j is visible to token i iff j <= shift + i (causal), j < kv
};

__device__ __forceinline__ ReqView request_view(const PagedArgs &g, int r) {
    ReqView v;
    const long long T = g.T;
    const long long q0 = min((long long)max(g.cu[r], 0), T);
    const long long q1 = max(min((long long)g.cu[r + 1], T), q0);
    v.q0 = (int)q0, v.n = (int)(q1 - q0);
    const long long room = (long long)g.W << g.page_shift;
    v.kv = (int)min((long long)max(g.kv_lens[r], 0), room);
    v.shift = g.causal ? v.kv - v.n : 2147483647 - v.n;
    return v;
}
// keys that the last token of a tile sees, i.e. how far the tile has to read
__device__ __forceinline__ int keys_until(const ReqView &v, int last_token) {
    const int lim = min(v.shift + last_token + 1, v.kv);
    return max(lim, 0);
}

// Tiles of ROWS consecutive packed rows (a token's heads may be cut), KEYS keys per step.
template <int ROWS_, int KEYS>
struct PackedRows {
    static constexpr int ROWS = ROWS_;
    // token of the request and head of the group in `row` of a tile; false: the row is not in use
    static __device__ __forceinline__ bool place(const PagedArgs &g, const ReqView &v, int tile, int row, int &tok, int &j) {
        const long long packed = (long long)tile * ROWS + row;
        tok = (int)min(packed / g.group, (long long)v.n);
        j = (int)(packed % g.group);
        return tok < v.n;
    }
    static __device__ __forceinline__ int tiles(const PagedArgs &g, const ReqView &v) {
        return (int)(((long long)v.n * g.group + ROWS - 1) / ROWS);
    }
    static __device__ __forceinline__ int steps(const PagedArgs &g, const ReqView &v, int tile) {
        const long long last_row = min((long long)(tile + 1) * ROWS, (long long)v.n * g.group) - 1;
        const int keys = keys_until(v, (int)(last_row / g.group));
        return max((keys + KEYS - 1) / KEYS, 1);
    }
    static __device__ __forceinline__ long long head_steps(const PagedArgs &g, const ReqView &v) {
        long long s = 0;
        const int n = tiles(g, v);
        for (int t = 0; t < n; ++t) s += steps(g, v, t);
        return s;
    }
};

// Pairs of 128-row tiles of whole tokens (128 / group tokens each), KEYS keys per step.
template <int KEYS>
struct TokenTiles {
    static constexpr int ROWS = 256;
    static __device__ __forceinline__ int tokens(const PagedArgs &g) { return 128 / g.group; }  // of one of the two
    static __device__ __forceinline__ bool place(const PagedArgs &g, const ReqView &v, int tile, int row, int &tok, int &j) {
        const int r = row & 127, t = r / g.group, n = tokens(g);
        tok = (2 * tile + (row >> 7)) * n + t;
        j = r - t * g.group;
        return t < n && tok < v.n;
    }
    static __device__ __forceinline__ int tiles(const PagedArgs &g, const ReqView &v) {
        const int n = 2 * tokens(g);
        return (v.n + n - 1) / n;
    }
    static __device__ __forceinline__ int steps(const PagedArgs &g, const ReqView &v, int tile) {
        const int last = min((tile + 1) * 2 * tokens(g), v.n) - 1;
        return max((keys_until(v, last) + KEYS - 1) / KEYS, 1);
    }
    static __device__ __forceinline__ long long head_steps(const PagedArgs &g, const ReqView &v) {
        long long s = 0;
        const int n = tiles(g, v);
        for (int t = 0; t < n; ++t) s += steps(g, v, t);
        return s;
    }
};

// A CTA's place in the list of items.
struct WorkPos {
    int req, head, tile;
    int step;          // first step of the current item that is this CTA's
    long long left;    // steps this CTA still has to take
    long long base;    // global number of the current item's first step
    long long total;   // U
    int ctas;          // CTAs that share the work
};

// Finds the CTA's first item.  Called by all threads of the CTA (block barriers inside); `scratch` holds
// 34 long longs plus one WorkPos in shared memory.
template <typename TL>
__device__ __forceinline__ bool find_work(const PagedArgs &g, WorkPos &out, long long *scratch) {
    const int nt = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = nt >> 5;
    WorkPos *found = reinterpret_cast<WorkPos *>(scratch + 34);
    const int per = (g.B + nt - 1) / nt;
    const int r0 = min(tid * per, g.B), r1 = min(r0 + per, g.B);
    long long mine = 0;
    for (int r = r0; r < r1; ++r) mine += TL::head_steps(g, request_view(g, r)) * g.Hkv;
    long long inc = mine;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const long long a = __shfl_up_sync(0xFFFFFFFFu, inc, s);
        if (lane >= s) inc += a;
    }
    if (lane == 31) scratch[warp] = inc;
    if (tid == 0) found->req = -1;
    __syncthreads();
    long long before = 0, total = 0;
    for (int w = 0; w < nw; ++w) {
        if (w < warp) before += scratch[w];
        total += scratch[w];
    }
    before += inc - mine;
    int ctas = (int)gridDim.x;
    const long long most = (total + g.min_steps - 1) / g.min_steps;
    if (most < ctas) ctas = (int)most;
    const int c = (int)blockIdx.x;
    if (c < ctas) {
        const long long u0 = total * c / ctas, u1 = total * (c + 1) / ctas;
        if (u0 >= before && u0 < before + mine) {  // one thread: the one whose requests hold step u0
            long long at = before;
            for (int r = r0; r < r1; ++r) {
                const ReqView v = request_view(g, r);
                const long long per_head = TL::head_steps(g, v);
                const long long all = per_head * g.Hkv;
                if (u0 >= at + all) {
                    at += all;
                    continue;
                }
                const int head = (int)((u0 - at) / per_head);
                at += per_head * head;
                int tile = 0;
                while (true) {
                    const int s = TL::steps(g, v, tile);
                    if (u0 < at + s) break;
                    at += s;
                    ++tile;
                }
                found->req = r, found->head = head, found->tile = tile;
                found->step = (int)(u0 - at);
                found->left = u1 - u0;
                found->base = at;
                found->total = total;
                found->ctas = ctas;
                break;
            }
        }
    }
    __syncthreads();
    out = *found;
    return out.req >= 0;
}

// Moves on to the next item of the list; false behind the last one.
template <typename TL>
__device__ __forceinline__ bool next_item(const PagedArgs &g, WorkPos &w, ReqView &v) {
    w.base += TL::steps(g, v, w.tile);
    w.step = 0;
    if (++w.tile < TL::tiles(g, v)) return true;
    w.tile = 0;
    if (++w.head < g.Hkv) return true;
    w.head = 0;
    while (++w.req < g.B) {
        v = request_view(g, w.req);
        if (v.n > 0) return true;
    }
    return false;
}

// The CTA that takes global step x.
__device__ __forceinline__ int cta_of_step(const WorkPos &w, long long x) {
    return (int)(((x + 1) * w.ctas - 1) / w.total);
}

// Floats of one partial result: ROWS x D numerators, then ROWS maxima and ROWS sums.
template <int ROWS, int D>
constexpr size_t kPartFloats = (size_t)ROWS * D + 2 * ROWS;

// Joins the partial results of cut items (kernel launched behind either schedule).
template <int DT, int D, typename TL>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedArgs g) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const PartialItem it = g.meta[blockIdx.x];
    if (it.last < 0) return;
    const ReqView v = request_view(g, it.req);
    const int lane = threadIdx.x & 31;
    constexpr int ROWS = TL::ROWS;
    const int row = blockIdx.y * 4 + (threadIdx.x >> 5);
    int tok, j;
    if (!TL::place(g, v, it.tile, row, tok, j)) return;
    const int c0 = (int)blockIdx.x, n = it.last - c0 + 1;
    // part i: the CTA that starts the item keeps it in its second slot, the following ones in their first
    auto part = [&](int i) { return g.part + ((size_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * kPartFloats<ROWS, D>; };
    float top = -INFINITY;
    for (int i = lane; i < n; i += 32) top = fmaxf(top, part(i)[(size_t)ROWS * D + row]);
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
    const float base = top == -INFINITY ? 0.f : top;
    constexpr int PER = D / 32;
    float acc[PER] = {}, sum = 0.f;
    for (int i0 = 0; i0 < n; i0 += 32) {
        float wt = 0.f, l = 0.f;
        if (i0 + lane < n) {
            const float *p = part(i0 + lane);
            wt = exp2f(p[(size_t)ROWS * D + row] - base);
            l = p[(size_t)ROWS * D + ROWS + row];
        }
        const int m = min(32, n - i0);
#pragma unroll 4
        for (int i = 0; i < m; ++i) {
            const float w = __shfl_sync(0xFFFFFFFFu, wt, i);
            sum = fmaf(w, __shfl_sync(0xFFFFFFFFu, l, i), sum);
            const float *p = part(i0 + i) + (size_t)row * D + lane * PER;
            if constexpr (PER == 4) {
                const float4 x = *reinterpret_cast<const float4 *>(p);
                acc[0] = fmaf(w, x.x, acc[0]), acc[1] = fmaf(w, x.y, acc[1]);
                acc[2] = fmaf(w, x.z, acc[2]), acc[3] = fmaf(w, x.w, acc[3]);
            } else {
                const float2 x = *reinterpret_cast<const float2 *>(p);
                acc[0] = fmaf(w, x.x, acc[0]), acc[1] = fmaf(w, x.y, acc[1]);
            }
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    const int head = it.head * g.group + j;
    char *o = g.o + 2 * (((long long)v.q0 + tok) * g.o_st + head * g.o_sh + lane * PER);
    if constexpr (PER == 4)
        *reinterpret_cast<uint2 *>(o) = make_uint2(Pack16<DT>::pack(acc[0] * inv, acc[1] * inv), Pack16<DT>::pack(acc[2] * inv, acc[3] * inv));
    else
        *reinterpret_cast<uint32_t *>(o) = Pack16<DT>::pack(acc[0] * inv, acc[1] * inv);
}

// Launches the join behind the kernel last launched on the stream; its blocks may be scheduled while
// that kernel drains and wait for its results on the device.
template <int DT, int D, typename TL>
int launch_join(const PagedArgs &g, unsigned ctas, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, TL::ROWS / 4);
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, paged_join_kernel<DT, D, TL>, g);
}

}  // namespace deca
