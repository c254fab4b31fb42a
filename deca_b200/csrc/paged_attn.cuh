// What the two paged-attention schedules share: the device's view of the arguments, the list of work
// items, its division among the CTAs and the layout of partial results.
//
// Lengths live on the device, so the division is made there.  An item is one tile of query rows of one
// request and key head; row i of a tile packs token i / group and query head i % group of the key head, so
// all rows of an item read the same keys.  An item costs as many steps as it has key tiles (one at least: a
// row that sees no key is still written), and its start and end as much as a few more (kItemSteps), which come
// first.  With U steps in all and G CTAs, CTA c takes the steps [U c / G, U (c + 1) / G) of the concatenated
// items: every CTA gets the same share, whatever the lengths are.  An item that is cut leaves one partial result
// per CTA (fp32 numerators, maximum and sum per row); they are joined in the order of the keys, so results do not
// depend on timing.
#pragma once

#include "ptx.cuh"
#include "tmap.cuh"

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
    int tile_tokens;       // TokenTiles: whole tokens in 128 rows
    int k_heads, v_heads;  // 0 where all key heads lie at the same place (a head stride of zero), else 1
    int page_shift;
    int causal;
    float sl2;  // scale * log2 e
    int min_steps;  // fewest steps worth a CTA of their own
    int max_parts;  // most CTAs per request and key head, on average
    float *part;    // partial results, 2 per CTA
    struct PartialItem *meta;     // one per CTA (tiles)
    unsigned long long *flags;    // 2 per CTA (rows): `tag` where the partial result is complete
    unsigned long long tag;       // this launch's
    DeviceStatus *status;
};

// The item that starts in a CTA's range and ends in a later one's; `last` < 0: none.
struct PartialItem {
    int last;        // the CTA that ends it
    int head, tile;
    int q0, n;       // of its request
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
    // Device time without / with 2 / with 4 / with 6 steps for an item's start and end: 64 requests of 1000 .. 8191 keys
    // (D = 128) 210 / 204 / 202 / 203 us, 200 of 1 .. 8000 keys 516 / 497 / 488 / 491.
    static constexpr int kItemSteps = 4;
    // token of the request and head of the group in `row` of a tile; false: the row is not in use
    static __device__ __forceinline__ bool place(const PagedArgs &g, int n, int tile, int row, int &tok, int &j) {
        const unsigned long long packed = (unsigned long long)tile * ROWS + row;
        const unsigned long long t = packed / (unsigned)g.group;
        tok = (int)min(t, (unsigned long long)n);
        j = (int)(packed - t * (unsigned)g.group);
        return tok < n;
    }
    static __device__ __forceinline__ int tiles(const PagedArgs &g, const ReqView &v) {
        return (int)(((unsigned long long)v.n * (unsigned)g.group + ROWS - 1) / ROWS);
    }
    // the last token of a tile; the division only where more tiles follow
    static __device__ __forceinline__ int last_token(const PagedArgs &g, const ReqView &v, int tile) {
        const unsigned long long end = (unsigned long long)(tile + 1) * ROWS;
        if (end >= (unsigned long long)v.n * (unsigned)g.group) return v.n - 1;
        return (int)((end - 1) / (unsigned)g.group);
    }
    static __device__ __forceinline__ int steps(const PagedArgs &g, const ReqView &v, int tile) {
        return max((keys_until(v, last_token(g, v, tile)) + KEYS - 1) / KEYS, 1);
    }
    static __device__ __forceinline__ long long head_steps(const PagedArgs &g, const ReqView &v) {
        const int n = tiles(g, v);
        long long s = (long long)n * kItemSteps;
        for (int t = 0; t < n; ++t) s += steps(g, v, t);
        return s;
    }
};

// Pairs of 128-row tiles of whole tokens (128 / group tokens each), KEYS keys per step.
template <int KEYS>
struct TokenTiles {
    static constexpr int ROWS = 256;
    // Device time without / with 1 / 2 / 3 / 4 steps (at D = 64 with a slower exponential than today's): 9 requests of 188 .. 700 tokens and up to 5000 keys (D = 64)
    // 187 / 151 / 134 / 139 / 142 us, 20 of up to 700 tokens (D = 128) 362 / 302 / 290 / 294 / 300, one of 8192 tokens
    // 547 / 507 / 488 / 494 / 501, 4 of 4096 with equal heads 342 / 329 / 332 / 319 / 324.
    static constexpr int kItemSteps = 2;
    static __device__ __forceinline__ int tokens(const PagedArgs &g) { return g.tile_tokens; }  // of one of the two
    static __device__ __forceinline__ bool place(const PagedArgs &g, int n, int tile, int row, int &tok, int &j) {
        const int r = row & 127, t = r / g.group;
        tok = (2 * tile + (row >> 7)) * tokens(g) + t;
        j = r - t * g.group;
        return t < tokens(g) && tok < n;
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
        const int n = tiles(g, v);
        long long s = (long long)n * kItemSteps;
        for (int t = 0; t < n; ++t) s += steps(g, v, t);
        return s;
    }
};

// A CTA's place in the list of items.
struct WorkPos {
    int req, head, tile;
    int step;  // first step of the current item that is this CTA's
    int left;  // steps this CTA still has to take, starts of later items included
};
// The CTA's range in the list; kept in shared memory, read where an item is cut.
struct WorkShare {
    long long end, total;  // one past its last step; steps in all
    int ctas;              // CTAs that share the work
    WorkPos first;
    long long warp_sum[32];
};

// Finds the CTA's first item.  Called by all threads of the CTA (block barriers inside); `costs` is shared
// memory for `room` requests' costs, free afterwards.
template <typename TL>
__device__ __forceinline__ bool find_work(const PagedArgs &g, WorkPos &out, WorkShare *share, unsigned long long *costs, int room) {
    const int nt = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = nt >> 5;
    auto cost_of = [&](int r) { return (unsigned long long)(TL::head_steps(g, request_view(g, r)) * g.Hkv); };
    // side by side through the requests' lengths, then each thread sums the costs of neighbours
    for (int r = tid; r < min(g.B, room); r += nt) costs[r] = cost_of(r);
    if (tid == 0) share->first.req = -1;
    __syncthreads();
    const int per = (g.B + nt - 1) / nt;
    const int r0 = min(tid * per, g.B), r1 = min(r0 + per, g.B);
    auto cost_at = [&](int r) { return r < room ? costs[r] : cost_of(r); };
    unsigned long long mine = 0;
    for (int r = r0; r < r1; ++r) mine += cost_at(r);
    unsigned long long inc = mine;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const unsigned long long a = __shfl_up_sync(0xFFFFFFFFu, inc, s);
        if (lane >= s) inc += a;
    }
    if (lane == 31) share->warp_sum[warp] = (long long)inc;
    __syncthreads();
    unsigned long long before = 0, total = 0;
    for (int w = 0; w < nw; ++w) {
        if (w < warp) before += share->warp_sum[w];
        total += share->warp_sum[w];
    }
    before += inc - mine;
    const unsigned long long most = min((total + g.min_steps - 1) / (unsigned)g.min_steps,
                                        (unsigned long long)g.B * (unsigned)g.Hkv * (unsigned)g.max_parts);
    const unsigned ctas = most < gridDim.x ? (unsigned)most : gridDim.x, c = blockIdx.x;
    if (c < ctas) {
        const unsigned long long u0 = total * c / ctas;
        if (u0 >= before && u0 < before + mine) {  // one thread: the one whose requests hold step u0
            unsigned long long at = before;
            int r = r0;
            for (; u0 >= at + cost_at(r); ++r) at += cost_at(r);
            const ReqView v = request_view(g, r);
            const unsigned long long per_head = cost_at(r) / (unsigned)g.Hkv;
            const int head = (int)((u0 - at) / per_head);
            at += per_head * head;
            int tile = 0;
            for (int s; u0 >= at + (s = TL::kItemSteps + TL::steps(g, v, tile)); ++tile) at += s;
            const unsigned long long u1 = total * (c + 1) / ctas;
            at += TL::kItemSteps;
            const unsigned long long from = max(u0, at);  // of a range that begins in an item's start the item is whole
            share->first.req = from < u1 ? r : -1, share->first.head = head, share->first.tile = tile;
            share->first.step = (int)(from - at);
            share->first.left = (int)min(u1 - from, 2147483647ull);
            share->end = (long long)u1;
            share->total = (long long)total;
            share->ctas = (int)ctas;
        }
    }
    __syncthreads();
    out = share->first;
    return out.req >= 0;
}

// Few items (at most half as many as CTAs, of at most 32 requests): instead of an equal run of steps each CTA gets
// one part of one item, so that none pays the start and end of two.  Items are cut into parts of at most C
// steps, C = steps / (CTAs - items) rounded up, which needs no more parts than CTAs.  Every warp finds its CTA's part
// by itself (lane r holds request r).  Returns 0 where there are too many items, 1 with a part, -1 without.
template <typename TL>
__device__ __forceinline__ int find_part(const PagedArgs &g, WorkPos &w, ReqView &v, int &part, int &parts) {
    if (g.B > 32) return 0;
    const int lane = threadIdx.x & 31;
    ReqView mine = {0, 0, 0, 0};
    int tiles = 0;
    unsigned long long steps = 0;
    if (lane < g.B) {
        mine = request_view(g, lane);
        tiles = TL::tiles(g, mine);
        if (2ll * tiles * g.Hkv > (int)gridDim.x) tiles = (int)gridDim.x;  // too many: said below
        for (int t = 0; t < tiles; ++t) steps += TL::steps(g, mine, t);
    }
    unsigned long long total = steps;
    int items = tiles;
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) {
        total += __shfl_xor_sync(0xFFFFFFFFu, total, s);
        items += __shfl_xor_sync(0xFFFFFFFFu, items, s);
    }
    total *= (unsigned)g.Hkv;
    if (2ll * items * g.Hkv > (int)gridDim.x) return 0;
    if (items == 0) return -1;
    items *= g.Hkv;
    const unsigned room = gridDim.x - (unsigned)items;
    const int most = (int)max((total + room - 1) / room, (unsigned long long)g.min_steps);
    auto parts_of = [&](const ReqView &q, int t) { return (TL::steps(g, q, t) + most - 1) / most; };
    int count = 0;  // parts of one key head of this lane's request
    for (int t = 0; t < tiles; ++t) count += parts_of(mine, t);
    int end = count * g.Hkv;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int a = __shfl_up_sync(0xFFFFFFFFu, end, s);
        if (lane >= s) end += a;
    }
    const int at = (int)blockIdx.x - (end - count * g.Hkv);  // the CTA's place among this lane's parts
    const unsigned owner = __ballot_sync(0xFFFFFFFFu, at >= 0 && at < count * g.Hkv);
    if (owner == 0) return -1;
    const int r = __ffs((int)owner) - 1;
    v.q0 = __shfl_sync(0xFFFFFFFFu, mine.q0, r), v.n = __shfl_sync(0xFFFFFFFFu, mine.n, r);
    v.kv = __shfl_sync(0xFFFFFFFFu, mine.kv, r), v.shift = __shfl_sync(0xFFFFFFFFu, mine.shift, r);
    const int per_head = __shfl_sync(0xFFFFFFFFu, count, r);
    part = __shfl_sync(0xFFFFFFFFu, at, r);
    w.req = r, w.head = part / per_head, w.tile = 0;
    part -= w.head * per_head;
    for (; part >= (parts = parts_of(v, w.tile)); ++w.tile) part -= parts;
    const unsigned long long all = (unsigned)TL::steps(g, v, w.tile);
    w.step = (int)(all * (unsigned)part / (unsigned)parts);
    w.left = (int)(all * (unsigned)(part + 1) / (unsigned)parts) - w.step;
    return 1;
}

// Moves on to the next item of the list; false where the CTA's range ends before its first step.
template <typename TL>
__device__ __forceinline__ bool next_item(const PagedArgs &g, WorkPos &w, ReqView &v) {
    w.left -= TL::kItemSteps;
    if (w.left <= 0) return false;
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

// The CTA that takes step x: the last c with total * c / ctas <= x.
__device__ __forceinline__ int cta_of(const WorkShare *share, long long x) {
    return (int)(((unsigned long long)(x + 1) * (unsigned)share->ctas - 1) / (unsigned long long)share->total);
}

// Floats of one partial result: ROWS x D numerators, then ROWS maxima and ROWS sums.
template <int ROWS, int D>
constexpr size_t kPartFloats = (size_t)ROWS * D + 2 * ROWS;

// One row of a cut item from its n parts, by one warp.  Lane i reads the statistics of part i (of 32) while the
// numerators of BATCH parts are on their way.  part(i): the i-th part; acc: D / 32 columns of this lane.
template <int ROWS, int D, int BATCH, typename Part>
__device__ __forceinline__ void join_row(Part part, int n, int row, int lane, float (&acc)[D / 32], float &sum) {
    constexpr int PER = D / 32;
    float top = -INFINITY;
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < PER; ++k) acc[k] = 0.f;
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += 32) {
        float m = -INFINITY, l = 0.f;
        if (i0 + lane < n) {
            const float *p = part(i0 + lane) + (size_t)ROWS * D + row;
            m = __ldcg(p), l = __ldcg(p + ROWS);
        }
        float wt = 0.f;
#pragma unroll 1
        for (int b0 = 0; b0 < 32 && i0 + b0 < n; b0 += BATCH) {
            float x[BATCH][PER];
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
#pragma unroll
                for (int k = 0; k < PER; ++k) x[b][k] = 0.f;
                if (i0 + b0 + b < n) {
                    const float *p = part(i0 + b0 + b) + (size_t)row * D;
                    if constexpr (PER == 4) {
                        const float4 v = __ldcg(reinterpret_cast<const float4 *>(p) + lane);
                        x[b][0] = v.x, x[b][1] = v.y, x[b][2] = v.z, x[b][3] = v.w;
                    } else {
                        const float2 v = __ldcg(reinterpret_cast<const float2 *>(p) + lane);
                        x[b][0] = v.x, x[b][1] = v.y;
                    }
                }
            }
            if (b0 == 0) {  // weights of these 32 parts, and what came before brought to the same maximum
                float up = m;
#pragma unroll
                for (int s = 16; s >= 1; s >>= 1) up = fmaxf(up, __shfl_xor_sync(0xFFFFFFFFu, up, s));
                up = fmaxf(up, top);
                const float base = up == -INFINITY ? 0.f : up;
                wt = exp2f(m - base);
                const float old = exp2f(top - base);
                top = up;
                float part_sum = wt * l;
#pragma unroll
                for (int s = 16; s >= 1; s >>= 1) part_sum += __shfl_xor_sync(0xFFFFFFFFu, part_sum, s);
                sum = fmaf(sum, old, part_sum);
#pragma unroll
                for (int k = 0; k < PER; ++k) acc[k] *= old;
            }
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                const float w = __shfl_sync(0xFFFFFFFFu, wt, (b0 + b) & 31);
                if (i0 + b0 + b >= n) continue;
#pragma unroll
                for (int k = 0; k < PER; ++k) acc[k] = fmaf(w, x[b][k], acc[k]);
            }
        }
    }
}

template <int DT, int D>
__device__ __forceinline__ void store_joined(char *row, int lane, const float (&acc)[D / 32], float sum) {
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    if constexpr (D == 128)
        *reinterpret_cast<uint2 *>(row + lane * 8) =
            make_uint2(Pack16<DT>::pack(acc[0] * inv, acc[1] * inv), Pack16<DT>::pack(acc[2] * inv, acc[3] * inv));
    else
        *reinterpret_cast<uint32_t *>(row + lane * 4) = Pack16<DT>::pack(acc[0] * inv, acc[1] * inv);
}

// Joins the items that the tiles' CTAs have cut: a kernel behind theirs.
constexpr int kJoinThreads = 256;
template <int DT, int D, typename TL>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedArgs g) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const PartialItem it = g.meta[blockIdx.x];
    if (it.last < 0) return;
    const int lane = threadIdx.x & 31, c0 = (int)blockIdx.x;
    // part i: the CTA that starts the item keeps it in its second slot, the following ones in their first
    auto part = [&](int i) { return g.part + ((size_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * kPartFloats<TL::ROWS, D>; };
    const int warp = threadIdx.x >> 5, warps = kJoinThreads / 32;
    if (it.last == c0 + 1) {
        // two parts, the usual case: four rows of a warp with all their loads in flight
        constexpr int R = 4, PER = D / 32;
        const float *p0 = part(0), *p1 = part(1);
        for (int row0 = (blockIdx.y * warps + warp) * R; row0 < TL::ROWS; row0 += gridDim.y * warps * R) {
            float m0[R], m1[R], l0[R], l1[R], x0[R][PER], x1[R][PER];
            auto numerators = [&](const float *p, int row, float (&x)[PER]) {
                if constexpr (PER == 4) {
                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(p + (size_t)row * D) + lane);
                    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
                } else {
                    const float2 v = __ldcg(reinterpret_cast<const float2 *>(p + (size_t)row * D) + lane);
                    x[0] = v.x, x[1] = v.y;
                }
            };
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const size_t at = (size_t)TL::ROWS * D + row0 + i;
                m0[i] = __ldcg(p0 + at), l0[i] = __ldcg(p0 + at + TL::ROWS);
                m1[i] = __ldcg(p1 + at), l1[i] = __ldcg(p1 + at + TL::ROWS);
                numerators(p0, row0 + i, x0[i]);
                numerators(p1, row0 + i, x1[i]);
            }
#pragma unroll
            for (int i = 0; i < R; ++i) {
                int tok, j;
                if (!TL::place(g, it.n, it.tile, row0 + i, tok, j)) continue;
                const float top = fmaxf(m0[i], m1[i]), base = top == -INFINITY ? 0.f : top;
                const float w0 = exp2f(m0[i] - base), w1 = exp2f(m1[i] - base);
                float acc[PER];
#pragma unroll
                for (int k = 0; k < PER; ++k) acc[k] = fmaf(w0, x0[i][k], w1 * x1[i][k]);
                store_joined<DT, D>(g.o + 2 * (((long long)it.q0 + tok) * g.o_st + (long long)(it.head * g.group + j) * g.o_sh), lane, acc,
                                    fmaf(w0, l0[i], w1 * l1[i]));
            }
        }
        return;
    }
    for (int row = blockIdx.y * warps + warp; row < TL::ROWS; row += gridDim.y * warps) {
        int tok, j;
        if (!TL::place(g, it.n, it.tile, row, tok, j)) continue;
        float acc[D / 32], sum;
        join_row<TL::ROWS, D, 4>(part, it.last - c0 + 1, row, lane, acc, sum);
        store_joined<DT, D>(g.o + 2 * (((long long)it.q0 + tok) * g.o_st + (long long)(it.head * g.group + j) * g.o_sh), lane, acc, sum);
    }
}

// Tensor maps of the caches, (d, row of the page, key head, page), with boxes of 64 columns and the rows of a page
// or `keys`, whichever is less.
inline int make_cache_maps(CUtensorMap *tmK, CUtensorMap *tmV, int dtype, int D, int keys, const PagedArgs &g) {
    const uint64_t page = 1ull << g.page_shift;
    const uint32_t box[4] = {64, (uint32_t)(page < (uint64_t)keys ? page : keys), 1, 1};
    const uint64_t kd[4] = {(uint64_t)D, page, g.k_heads ? (uint64_t)g.Hkv : 1, (uint64_t)g.num_pages};
    const uint64_t vd[4] = {(uint64_t)D, page, g.v_heads ? (uint64_t)g.Hkv : 1, (uint64_t)g.num_pages};
    const uint64_t ks[3] = {(uint64_t)g.k_sr * 2, (uint64_t)g.k_sh * 2, (uint64_t)g.k_sp * 2};
    const uint64_t vs[3] = {(uint64_t)g.v_sr * 2, (uint64_t)g.v_sh * 2, (uint64_t)g.v_sp * 2};
    if (int rc = make_tmap_16bit(tmK, dtype, g.k, 4, kd, ks, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
    return make_tmap_16bit(tmV, dtype, g.v, 4, vd, vs, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Lets the next kernel of the stream be scheduled while this one drains (it waits for the results itself).
__device__ __forceinline__ void allow_next_kernel() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launches the join behind the kernel last launched on the stream; its blocks may be scheduled while
// that kernel drains and wait for its results on the device.
template <int DT, int D, typename TL>
int launch_join(const PagedArgs &g, unsigned ctas, unsigned blocks, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, blocks);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, paged_join_kernel<DT, D, TL>, g);
}

}  // namespace deca
