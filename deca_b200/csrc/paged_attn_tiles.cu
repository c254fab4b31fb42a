// Paged attention for many query rows per request (prompt chunks): tcgen05 tiles over the paged cache.
//
// The roles and barriers are those of the dense persistent schedule (fa_fwd3_f16.cu): one CTA per SM, a
// TMA producer, one MMA-issuing thread, two groups of four softmax warps with a 128-row tile each, a
// relay warp; S and P in tensor memory, P consumed from there; the running maximum moves only when a row
// sum exceeds 2^8.  What differs:
//   * An item is a pair of Q tiles of one request and key head, 128 / group whole tokens times the group's
//     heads each: all query heads of a key head share its K and V tiles, and a short chunk still fills
//     rows.  A Q tile is one box of a four-dimensional tensor map (d, head in group, key head, token).
//   * A K or V tile of 128 keys is gathered through the block table with one box per page (or half of a
//     256-row page) and 64 columns; each lane of the producer warp issues its own box.
//   * The CTA takes a contiguous range of steps of the item list (paged_attn.cuh) instead of whole items;
//     an item that is cut leaves fp32 partial results that a second kernel joins.
//   * The relay makes the V tiles of an item's end safe before they are multiplied: rows behind the last
//     key become zero, whatever the cache holds there; an element that is not finite in a key that only
//     some of the item's rows see is replaced by zero and noted (first such key of each column and
//     kind), and the epilogue gives it to the rows that do see it.
// Bound by the chain of a step (scores, exponentials, product): 2.2 us at D = 128 and 1.8 - 1.9 at D = 64 for 2 x 128 x 128
// scores; of the 3550 clocks at D = 128 the softmax of a tile takes 1480 and its MMAs 1500 up to the next scores' arrival,
// the two tiles' MMAs following each other.  Device time: 2 x 2048 tokens behind 6144 (fp16, D = 128, 4 query
// heads a key head) 420 - 425 us = 1.14 PFLOPS (the dense persistent schedule: 1.09 sustained, 1.28 in isolated launches), 1 x 8192 485,
// 4 x 4096 with 16 equal heads 325 (D = 64: 258), a ragged batch of 9 at D = 64 127.
// Tried and slower: two warps per 32 rows (445 us on the first of these), an issuing thread per tile (567), P in
// columns of its own at D = 64, which tensor memory has room for, so that scores run ahead (6 % on the last); no gain:
// the next item's first scores issued before the last product (426).
#include <cuda.h>

#include "fa_softmax.cuh"
#include "paged_attn.cuh"
#include "tmap.cuh"

namespace deca {
namespace {

constexpr int kBr = 128;
constexpr int kBc = 128;
constexpr int kThreads = 352;  // TMA producer, MMA issuer, 2 x 4 softmax warps, relay
constexpr uint32_t kStageBytes = 8 * 4096;  // one 4 KB output panel per softmax warp
constexpr int kNone = 255;  // no key noted

using TL = TokenTiles<kBc>;

template <int D>
struct Layout {
    static constexpr int kStages = D == 128 ? 4 : 8;
    static constexpr uint32_t kQBytes = kBr * D * 2, kKVBytes = kBc * D * 2;
    static constexpr uint32_t kNotes = 2 * 3 * D;  // two items x (NaN, +inf, -inf) x column: a byte each
    static constexpr uint32_t q = 0;
    static constexpr uint32_t kv = q + 2 * kQBytes;
    static constexpr uint32_t stage = kv + kStages * kKVBytes;
    static constexpr uint32_t notes = stage + kStageBytes;
    static constexpr uint32_t share = notes + kNotes + 16;  // 16: flags of the two items' notes
    static constexpr uint32_t bars = share + (sizeof(WorkShare) + 15) / 16 * 16;
    static constexpr uint32_t bytes = bars + 8 * (2 * kStages + 11);
    static constexpr size_t smem = 1024 + bytes;
};

struct RingPos {
    int slot;
    uint32_t par;
};

// Exponentials of 32 scores against the maximum's term: packed to 16 bits, summed in fp32.  A masked score is -inf,
// its exponential exactly zero; a NaN reaches the sum.  All of them on the exp2 unit, at D = 64 too: with every fourth
// pair as a polynomial on the FMA pipe (which pays in the dense kernel) 9 ragged requests took 134 us instead of 128, 4 x 512
// tokens behind 8192 129 instead of 123, 4 x 4096 265 instead of 258.
template <int DT>
__device__ __forceinline__ void exp_chunk32(const uint32_t (&v)[32], uint64_t sl2x2, uint64_t nmsx2, uint64_t (&sum2)[2],
                                            uint32_t *pk) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float x0, x1;
        f32x2_unpack(f32x2_fma(f32x2_pack(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), sl2x2, nmsx2), x0, x1);
        const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
        sum2[i & 1] = f32x2_add(sum2[i & 1], f32x2_pack(p0, p1));
        pk[i] = Pack16<DT>::pack(p0, p1);
    }
}

__device__ __forceinline__ float max32(const uint32_t (&v)[32]) {
    float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 32; ++i) part[i & 3] = fmaxf(part[i & 3], __uint_as_float(v[i]));
    return fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
}

// Exponentials of the whole row into registers; returns their sum.  The next 32 columns are on their way from
// tensor memory while the current ones are processed.
template <int DT>
__device__ __forceinline__ float exp_row(uint32_t tS, float sl2, float ms, uint32_t (&pk)[kBc / 2]) {
    const uint64_t sl2x2 = f32x2_pack(sl2, sl2), nmsx2 = f32x2_pack(-ms, -ms);
    uint64_t sum2[2] = {0ull, 0ull};
    uint32_t v[2][32];
    tmem_ld_32x32b_x32(tS, v[0]);
    tmem_ld_wait_regs(v[0]);
#pragma unroll
    for (int c = 0; c < kBc / 32; ++c) {
        if (c + 1 < kBc / 32) tmem_ld_32x32b_x32(tS + (c + 1) * 32, v[(c + 1) & 1]);
        exp_chunk32<DT>(v[c & 1], sl2x2, nmsx2, sum2, &pk[c * 16]);
        if (c + 1 < kBc / 32) tmem_ld_wait_regs(v[(c + 1) & 1]);
    }
    float a0, a1, b0, b1;
    f32x2_unpack(sum2[0], a0, a1);
    f32x2_unpack(sum2[1], b0, b1);
    return (a0 + a1) + (b0 + b1);
}

// Puts -inf where the row does not see the key: `visible` leading columns of the tile stay.
__device__ __forceinline__ void mask_tile(uint32_t tS, int visible) {
#pragma unroll 1
    for (int c = 0; c < kBc / 32; ++c) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(tS + c * 32, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (c * 32 + i >= visible) v[i] = 0xFF800000u;
        tmem_st_32x32b_x32(tS + c * 32, v);
    }
    tmem_st_wait();
}

// One key tile of the online softmax for this thread's row; `sees`: the row belongs to a token and sees a key of this tile.
// A row sees a prefix of the keys, so one that sees nothing of a segment's first 32 keys sees nothing of it: m
// stays -inf, l and P zero.  Rows behind the request's last token hold other requests' queries or padding; they have
// no voice in the warp's vote, or what they hold would choose the pass, and with it the rounding, of the others.
// A row that sees keys while its maximum is still -inf (all its scores so far were) has no base to take exponentials
// against: its fast sum comes out infinite or NaN, and the second pass finds the maximum.
// There is one copy of the exponentials' straight-line code: masked tiles are masked in place before it, and the
// rare second pass is a loop.  The warps' roles share the instruction cache, and what falls out of it costs an
// item microseconds when it ends (with a copy for each case 4 us from the last product of an item to the first
// score of the next).
template <int DT, int D>
__device__ __forceinline__ void softmax_tile(uint32_t tS, uint32_t tO, float sl2, bool first, bool sees, float &m, float &l) {
    if (first) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(tS, v);
        tmem_ld_wait();
        m = max32(v);
    }
    {
        // held in registers until the vote: storing P overwrites the scores that a second pass would need
        uint32_t pk[kBc / 2];
        const float sum = exp_row<DT>(tS, sl2, sees ? m * sl2 : 0.f, pk);
        if (!__any_sync(0xFFFFFFFFu, sees && !(sum <= kFaSumLimit))) {
#pragma unroll
            for (int h = 0; h < kBc / 64; ++h) {
                uint32_t part[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) part[i] = pk[h * 32 + i];
                tmem_st_32x32b_x32(tS + h * 32, part);
            }
            tmem_st_wait();
            l += sum;
            return;
        }
    }
    float top = m;
#pragma unroll 1
    for (int c = 0; c < kBc / 32; ++c) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(tS + c * 32, v);
        tmem_ld_wait();
        top = fmaxf(top, max32(v));
    }
    const float alpha = m == -INFINITY ? 0.f : ex2_approx((m - top) * sl2);
    l *= alpha;
    m = top;
    if (!first) {
        // the product of the previous tile is complete: it was issued before this tile's scores
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(tO + c * 32, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
            tmem_st_32x32b_x32(tO + c * 32, v);
        }
    }
    // P of scores 64 c .. goes over columns that have been read
    const float ms = m == -INFINITY ? 0.f : m * sl2;
#pragma unroll 1
    for (int c = 0; c < kBc / 64; ++c) {
        uint32_t pk[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(tS + c * 64 + h * 32, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p0 = ex2_approx(fmaf(__uint_as_float(v[2 * i]), sl2, -ms));
                const float p1 = ex2_approx(fmaf(__uint_as_float(v[2 * i + 1]), sl2, -ms));
                l += p0 + p1;
                pk[h * 16 + i] = Pack16<DT>::pack(p0, p1);
            }
        }
        tmem_st_32x32b_x32(tS + c * 32, pk);
    }
    tmem_st_wait();
}

// Bit 15 or 31 is set where that half of a packed pair is an infinity or a NaN (other bits are noise).
template <int DT>
__device__ __forceinline__ uint32_t exponent_carry(uint32_t w) {
    return DT == DECA_F16 ? (w & 0x7C007C00u) + 0x04000400u : (w & 0x7F807F80u) + 0x00800080u;
}

template <int DT, int D>
__global__ void __launch_bounds__(kThreads, 1)
paged_tiles_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                   const __grid_constant__ CUtensorMap tmV, const PagedArgs g) {
    using L = Layout<D>;
    constexpr int kStages = L::kStages;
    constexpr uint32_t kKVBlock = kBc * 128;
    constexpr uint32_t kIdescQK = make_idesc_f16(DT, false, false, kBr, kBc);
    constexpr uint32_t kIdescPV = make_idesc_f16(DT, false, true, kBr, D);
    constexpr uint32_t kTmemCols = 512;  // S_A, S_B (128 each), O_A, O_B (D each)

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t *smem = smem_raw + (base - raw);
    const uint32_t sQ = base + L::q, sKV = base + L::kv;
    uint8_t *notes = smem + L::notes;
    volatile int *noted = reinterpret_cast<volatile int *>(smem + L::notes + L::kNotes);
    const uint32_t q_full = base + L::bars, q_free = q_full + 8u;
    auto kv_full = [&](int i) { return q_full + 8u * (2 + i); };
    auto kv_empty = [&](int i) { return q_full + 8u * (2 + kStages + i); };
    const uint32_t fixed0 = q_full + 8u * (2 + 2 * kStages);
    auto s_full = [&](int grp) { return fixed0 + 8u * grp; };
    auto p_full = [&](int grp) { return fixed0 + 8u * (2 + grp); };
    auto pv_done = [&](int grp) { return fixed0 + 8u * (4 + grp); };
    const uint32_t drain_bar = fixed0 + 8u * 6, slot_addr = fixed0 + 8u * 7;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem + (slot_addr - base));
    volatile uint32_t *abort_flag = tmem_slot + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tpt = TL::tokens(g), used = tpt * g.group;  // tokens and rows of a Q tile

    if (threadIdx.x == 0) g.meta[blockIdx.x].last = -1;
    WorkPos w;
    allow_next_kernel();
    WorkShare *share = reinterpret_cast<WorkShare *>(smem + L::share);
    ReqView v;
    int part_no = 0, n_parts = 0;  // > 0: this CTA has this one part of an item
    const int found = find_part<TL>(g, w, v, part_no, n_parts);
    if (found < 0) return;
    if (found == 0) {
        n_parts = 0;
        // the ring is free for the costs
        if (!find_work<TL>(g, w, share, reinterpret_cast<unsigned long long *>(smem + L::kv), (int)(kStages * L::kKVBytes / 8))) return;
        v = request_view(g, w.req);
    }

    // rows of the Q tiles that no token reaches stay zero
    for (int i = threadIdx.x; i < 2 * (D / 64) * (kBr - used) * 8; i += kThreads) {
        const int c = i & 7, row = used + (i >> 3) % (kBr - used), blk = (i >> 3) / (kBr - used);
        *reinterpret_cast<uint4 *>(smem + L::q + blk * 16384 + row * 128 + c * 16) = make_uint4(0, 0, 0, 0);
    }
    for (int i = threadIdx.x; i < (int)L::kNotes; i += kThreads) notes[i] = kNone;
    fence_proxy_async_smem();
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        noted[0] = noted[1] = 0;
        mbar_init(q_full, 1);
        mbar_init(q_free, 1);
        for (int i = 0; i < kStages; ++i) {
            mbar_init(kv_full(i), 1);
            mbar_init(kv_empty(i), 1);
        }
        for (int grp = 0; grp < 2; ++grp) {
            mbar_init(s_full(grp), 1);
            mbar_init(p_full(grp), 5);  // four softmax warps + the relay
            mbar_init(pv_done(grp), 1);
        }
        mbar_init(drain_bar, 1);
        fence_barrier_init();
        prefetch_tensormap(&tmQ);
        prefetch_tensormap(&tmK);
        prefetch_tensormap(&tmV);
    }
    if (warp == 1) {
        tmem_alloc(slot_addr, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    auto tS = [&](int grp) { return tmem_base + (uint32_t)(grp * kBc); };
    auto tO = [&](int grp) { return tmem_base + 2u * kBc + (uint32_t)(grp * D); };
    auto advance = [&](RingPos &p, int n) {
        p.slot += n;
        while (p.slot >= kStages) p.slot -= kStages, p.par ^= 1u;
    };
    auto wait_all = [&](uint32_t bar, uint32_t parity) {
        return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag)) != 0;
    };
    auto segment = [&](int &steps) {  // steps of the current item that are this CTA's
        steps = TL::steps(g, v, w.tile);
        return min(steps - w.step, w.left);
    };
    auto next = [&](int n) {
        w.left -= n;
        return w.left > 0 && n_parts == 0 && next_item<TL>(g, w, v);
    };
    // keys that the item reads, and the last one that all of its rows see
    auto item_keys = [&](int &kend, int &common) {
        const int first = w.tile * 2 * tpt;
        kend = keys_until(v, min(first + 2 * tpt, v.n) - 1);
        common = min(v.shift + first, v.kv - 1);
    };

    bool ok = true;
    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer
        RingPos rp{0, 0u};
        const int rows = min(1 << g.page_shift, kBc);       // of a box
        const int boxes = kBc / rows;                       // per 64 columns
        const int blk = lane / boxes, box = lane % boxes;
        const bool mine = lane < boxes * (D / 64);
        const uint32_t dst = sKV + blk * kKVBlock + box * rows * 128;
        int n_local = 0;
        while (true) {
            int steps;
            const int n = segment(steps);
            int kend, common;
            item_keys(kend, common);
            if (n_local > 0 && !wait_all(q_free, (uint32_t)((n_local - 1) & 1))) {
                if (lane == 0) report_detail(g.status, 0, 1, n_local);
                ok = false;
                break;
            }
            if (lane == 0) {
                mbar_arrive_expect_tx(q_full, 2u * (uint32_t)used * D * 2u);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int b = 0; b < D / 64; ++b)
                        tma_load_4d(sQ + t * L::kQBytes + b * 16384, &tmQ, b * 64, 0, w.head, v.q0 + (2 * w.tile + t) * tpt, q_full);
            }
            const int *table = g.table + w.req * g.table_stride;
            auto page_of = [&](int tile) {  // of this lane's box of a key tile; -1: behind the last key
                const long long key = (long long)tile * kBc + box * rows;
                if (!mine || key >= kend) return -1;
                const int p = table[key >> g.page_shift];
                return p >= 0 && p < g.num_pages ? p : (int)g.num_pages;  // a box outside the cache reads zeros
            };
            int page = page_of(w.step);
            for (int i = 0; i < n && ok; ++i) {
                const int tile = w.step + i;
                const int page_next = i + 1 < n ? page_of(tile + 1) : -1;
                const int row = (tile * kBc + box * rows) & ((1 << g.page_shift) - 1);
                const int live = min(max((kend - tile * kBc + rows - 1) / rows, 0), boxes);
#pragma unroll 1
                for (int kv = 0; kv < 2; ++kv) {
                    if (!wait_all(kv_empty(rp.slot), rp.par ^ 1u)) {
                        if (lane == 0) report_detail(g.status, 0, 2, i);
                        ok = false;
                        break;
                    }
                    if (lane == 0) mbar_arrive_expect_tx(kv_full(rp.slot), (uint32_t)(live * rows * D * 2));
                    __syncwarp();
                    if (page >= 0)
                        tma_load_4d(dst + rp.slot * L::kKVBytes, kv ? &tmV : &tmK, blk * 64, row,
                                    w.head * (kv ? g.v_heads : g.k_heads), page, kv_full(rp.slot));
                    advance(rp, 1);
                }
                page = page_next;
            }
            ++n_local;
            if (!ok || !next(n)) break;
        }
        // A wait that ran out lasted a second since this warp's last copy was issued, so none of its
        // copies is still in flight when the CTA leaves.
        if (!ok && lane == 0 && *abort_flag == 0) {
            *abort_flag = 1;
            report_timeout(g.status, 0x421u);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        if (lane == 0) {
            constexpr uint64_t kDescK = (uint64_t(16 >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
            constexpr uint64_t kDescV = (uint64_t((kKVBlock >> 4) & 0x3FFF) << 16) | (uint64_t(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
            const uint64_t q_desc = kDescK | (uint64_t)((sQ & 0x3FFFFu) >> 4);
            RingPos kp{0, 0u}, vp{1, 0u};
            uint32_t cnt = 0;  // key tiles handled so far
            int n_local = 0;
            while (ok) {
                int steps;
                const int n = segment(steps);
                if (!mbar_wait(q_full, (uint32_t)(n_local & 1), abort_flag) || !mbar_wait(kv_full(kp.slot), kp.par, abort_flag)) {
                    report_detail(g.status, 1, 3, n_local);
                    ok = false;
                    break;
                }
                // round j: the products of tile j (none in round -1) and the scores of tile j + 1
#pragma unroll 1
                for (int j = -1; j < n && ok; ++j) {
                    const uint64_t kdesc = kDescK | (uint64_t)(((sKV + kp.slot * L::kKVBytes) & 0x3FFFFu) >> 4);
                    const uint64_t vdesc = kDescV | (uint64_t)(((sKV + vp.slot * L::kKVBytes) & 0x3FFFFu) >> 4);
#pragma unroll
                    for (int grp = 0; grp < 2; ++grp) {
                        const uint32_t s_tmem = tS(grp), o_tmem = tO(grp);
                        if (j >= 0) {
                            // V_j and K_{j+1} have landed once p_full completes: the relay arrives there after them
                            if (!mbar_wait(p_full(grp), (cnt + (uint32_t)j) & 1u, abort_flag)) {
                                report_detail(g.status, 1, 5 + grp, j);
                                ok = false;
                                break;
                            }
                            tc_fence_after_sync();
#pragma unroll
                            for (int kk = 0; kk < kBc / 16; ++kk)  // O_grp (+)= P_grp V
                                umma_f16_ts(o_tmem, s_tmem + kk * 8, vdesc + kk * (2048 >> 4), kIdescPV, (j | kk) != 0 ? 1u : 0u);
                            if (j + 1 == n) umma_commit(pv_done(grp));  // the segment's O_grp is complete
                            if (grp == 1) umma_commit(kv_empty(vp.slot));
                        } else {
                            tc_fence_after_sync();
                        }
                        if (j + 1 < n) {
                            const uint64_t qd = q_desc + grp * (L::kQBytes >> 4);
#pragma unroll
                            for (int kd = 0; kd < D / 16; ++kd)  // S_grp = Q_grp K^T
                                umma_f16_ss(s_tmem, qd + (((kd / 4) * 16384 + (kd % 4) * 32) >> 4),
                                            kdesc + (((kd / 4) * kKVBlock + (kd % 4) * 32) >> 4), kIdescQK, kd != 0 ? 1u : 0u);
                            umma_commit(s_full(grp));
                            if (grp == 1) {
                                umma_commit(kv_empty(kp.slot));
                                if (j + 2 == n) umma_commit(q_free);  // the segment's last score MMA
                            }
                        }
                    }
                    if (j >= 0) advance(vp, 2);
                    if (j + 1 < n) advance(kp, 2);
                }
                cnt += (uint32_t)n;
                ++n_local;
                if (!ok || !next(n)) break;
            }
            if (!ok) {
                if (*abort_flag == 0) {
                    *abort_flag = 1;
                    report_timeout(g.status, 0x422u);
                }
                __shared__ uint32_t no_abort;
                no_abort = 0;
                umma_commit(drain_bar);
                (void)mbar_wait(drain_bar, 0, &no_abort);
            }
        }
        __syncwarp();
    } else if (warp == 10) {
        // ------------------------------------------------------------------ relay
        RingPos kp{0, 0u}, vp{1, 0u};
        uint32_t cnt = 0;
        int item = 0;
        uint32_t dirty = 0;  // bit b: the notes of buffer b are in use
        while (true) {
            int steps;
            const int n = segment(steps);
            int kend, common;
            item_keys(kend, common);
            const int buf = item & 1;
            advance(kp, 2);  // K_0: the issuer waits for it itself, together with Q
            for (int j = 0; j < n && ok; ++j) {
                const uint32_t t = cnt + (uint32_t)j;
                ok = wait_all(kv_full(vp.slot), vp.par) && (j + 1 >= n || wait_all(kv_full(kp.slot), kp.par));
                // an arrival must fall into the phase it is meant for: see the previous one complete
                for (int grp = 0; grp < 2 && ok && t > 0; ++grp) ok = wait_all(p_full(grp), (t - 1u) & 1u);
                if (!ok) {
                    if (lane == 0) report_detail(g.status, 10, 4, j);
                    break;
                }
                // The previous phase also means that both groups have left the epilogue of the item before
                // the last one, whose notes this buffer held.
                if (j == 0 && ((dirty >> buf) & 1u)) {
                    for (int i = lane; i < 3 * D; i += 32) notes[buf * 3 * D + i] = kNone;
                    if (lane == 0) noted[buf] = 0;
                    dirty &= ~(1u << buf);
                    __syncwarp();
                }
                const int key0 = (w.step + j) * kBc;
                if (key0 + kBc - 1 > common) {
                    uint8_t *tile = smem + L::kv + vp.slot * L::kKVBytes;
                    const int r0 = min(max(common + 1 - key0, 0), kBc), r1 = min(max(kend - key0, 0), kBc);
                    // an exponent of ones carries into the sign's place; eight loads are in flight
                    uint32_t seen = 0;
                    for (int i0 = r0 * 8 + lane; i0 < r1 * 8; i0 += 32 * 8 / (D / 64))
#pragma unroll
                        for (int k = 0; k < 8 / (D / 64); ++k)
#pragma unroll
                            for (int b = 0; b < D / 64; ++b) {
                                const int i = i0 + 32 * k;
                                const uint4 x = i < r1 * 8 ? *reinterpret_cast<const uint4 *>(tile + b * kKVBlock + i * 16) : make_uint4(0, 0, 0, 0);
                                seen |= exponent_carry<DT>(x.x) | exponent_carry<DT>(x.y) | exponent_carry<DT>(x.z) | exponent_carry<DT>(x.w);
                            }
                    const bool bad = (seen & 0x80008000u) != 0;
                    for (int i = r1 * 8 + lane; i < kBc * 8; i += 32)
#pragma unroll
                        for (int b = 0; b < D / 64; ++b)
                            *reinterpret_cast<uint4 *>(tile + b * kKVBlock + i * 16) = make_uint4(0, 0, 0, 0);
                    if (__any_sync(0xFFFFFFFFu, bad)) {
                        // column by column, keys in rising order: note the first of each kind
                        for (int d = lane; d < D; d += 32)
                            for (int r = r0; r < r1; ++r) {
                                uint16_t *x = reinterpret_cast<uint16_t *>(tile + (d >> 6) * kKVBlock + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4) + (d & 7) * 2);
                                constexpr uint32_t e = DT == DECA_F16 ? 0x7C00u : 0x7F80u;
                                const uint32_t bits = *x;
                                if ((bits & e) != e) continue;
                                const int kind = (bits & 0x7FFFu) != e ? 0 : (bits & 0x8000u) ? 2 : 1;
                                uint8_t *at = notes + (buf * 3 + kind) * D + d;
                                const int key = key0 + r - common - 1;
                                if (key < *at) *at = (uint8_t)key;
                                *x = 0;
                            }
                        dirty |= 1u << buf;
                        if (lane == 0) noted[buf] = 1;
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                if (lane < 2) mbar_arrive(p_full(lane));
                advance(vp, 2);
                if (j + 1 < n) advance(kp, 2);
            }
            cnt += (uint32_t)n;
            ++item;
            if (!ok || !next(n)) break;
        }
        if (!ok && lane == 0 && *abort_flag == 0) {
            *abort_flag = 1;
            report_timeout(g.status, 0x424u);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------------ softmax + epilogue
        const int grp = (warp - 2) >> 2;  // 0 = tile A, 1 = tile B
        const int q = warp & 3;           // tensor-memory lane quarter
        const int r = q * 32 + lane;
        const uint32_t lane_off = (uint32_t)(q * 32) << 16;
        const uint32_t tSg = tS(grp) + lane_off, tOg = tO(grp) + lane_off;
        uint8_t *panel = smem + L::stage + (warp - 2) * 4096;
        const float sl2 = g.sl2;
        uint32_t cnt = 0;
        int item = 0;
        while (true) {
            int steps;
            const int n = segment(steps);
            int kend, common;
            item_keys(kend, common);
            int tok, head;
            const bool live = TL::place(g, v.n, w.tile, grp * kBr + r, tok, head);
            const int lim = live ? min(v.shift + tok, v.kv - 1) : -1;
            const int lim_tile = min(v.shift + min((2 * w.tile + grp) * tpt, v.n), v.kv - 1);  // of the tile's first row
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < n; ++j) {
                if (!wait_all(s_full(grp), (cnt + (uint32_t)j) & 1u)) {
                    if (lane == 0 && q == 0) report_detail(g.status, 2 + grp, 7, j);
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                const int col0 = (w.step + j) * kBc;
                if (col0 + kBc - 1 > lim_tile) mask_tile(tSg, lim + 1 - col0);
                softmax_tile<DT, D>(tSg, tOg, sl2, j == 0, lim >= col0, m, l);
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(grp));
            }
            if (!ok) break;
            if (!wait_all(pv_done(grp), (uint32_t)(item & 1))) {
                if (lane == 0 && q == 0) report_detail(g.status, 2 + grp, 9, n);
                ok = false;
                break;
            }
            tc_fence_after_sync();
            cnt += (uint32_t)n;
            // ---- epilogue: through this warp's panel, so that eight lanes write 128 bytes of a row
            const bool whole = n == steps;
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            if (noted[item & 1] != 0) {
                // what was taken out of V goes to the rows that see it
                const uint8_t *note = notes + (item & 1) * 3 * D;
                const int seen = lim - common - 1;
#pragma unroll 1
                for (int b = 0; b < D / 32; ++b) {
                    uint32_t x[32];
                    tmem_ld_32x32b_x32(tOg + b * 32, x);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const uint8_t *at = note + b * 32 + i;
                        const bool up = at[D] <= seen, down = at[2 * D] <= seen;
                        if (up) x[i] = 0x7F800000u;
                        if (down) x[i] = 0xFF800000u;
                        if (at[0] <= seen || (up && down)) x[i] = 0x7FC00000u;
                    }
                    tmem_st_32x32b_x32(tOg + b * 32, x);
                }
                tmem_st_wait();
            }
            const int sub = lane >> 3, c8 = lane & 7;  // row within four, 16-byte chunk
            const uint32_t live_rows = __ballot_sync(0xFFFFFFFFu, live);
            if (whole) {
                const long long at = ((long long)v.q0 + tok) * g.o_st + (long long)(w.head * g.group + head) * g.o_sh;
#pragma unroll 1
                for (int b = 0; b < D / 64; ++b) {
                    uint32_t v0[32], v1[32];
                    tmem_ld_32x32b_x32(tOg + b * 64, v0);
                    tmem_ld_32x32b_x32(tOg + b * 64 + 32, v1);
                    tmem_ld_wait();
                    __syncwarp();  // the panel's previous rows have been read
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const uint32_t *x = c < 4 ? &v0[c * 8] : &v1[(c - 4) * 8];
                        uint32_t o[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            o[i] = Pack16<DT>::pack(__uint_as_float(x[2 * i]) * inv, __uint_as_float(x[2 * i + 1]) * inv);
                        *reinterpret_cast<uint4 *>(panel + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int row = i * 4 + sub;
                        const long long to = __shfl_sync(0xFFFFFFFFu, at, row);
                        if ((live_rows >> row) & 1u)
                            *reinterpret_cast<uint4 *>(g.o + 2 * (to + b * 64 + c8 * 8)) =
                                *reinterpret_cast<const uint4 *>(panel + row * 128 + ((c8 ^ (row & 7)) << 4));
                    }
                }
            } else {
                const bool starts = w.step == 0;
                float *part = g.part + ((size_t)blockIdx.x * 2 + (starts ? 1 : 0)) * kPartFloats<TL::ROWS, D>;
#pragma unroll 1
                for (int b = 0; b < D / 32; ++b) {
                    uint32_t v0[32];
                    tmem_ld_32x32b_x32(tOg + b * 32, v0);
                    tmem_ld_wait();
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        *reinterpret_cast<uint4 *>(panel + lane * 128 + ((c ^ (lane & 7)) << 4)) =
                            make_uint4(v0[4 * c], v0[4 * c + 1], v0[4 * c + 2], v0[4 * c + 3]);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int row = i * 4 + sub;
                        if ((live_rows >> row) & 1u)
                            *reinterpret_cast<uint4 *>(part + (size_t)(grp * kBr + q * 32 + row) * D + b * 32 + c8 * 4) =
                                *reinterpret_cast<const uint4 *>(panel + row * 128 + ((c8 ^ (row & 7)) << 4));
                    }
                }
                part[(size_t)TL::ROWS * D + grp * kBr + r] = m == -INFINITY ? m : m * sl2;
                part[(size_t)TL::ROWS * D + TL::ROWS + grp * kBr + r] = l;
                if (starts && threadIdx.x == 64) {
                    PartialItem it;
                    it.last = n_parts > 0 ? (int)blockIdx.x + n_parts - 1 : cta_of(share, share->end + (steps - n) - 1);
                    it.head = w.head, it.tile = w.tile, it.q0 = v.q0, it.n = v.n;
                    g.meta[blockIdx.x] = it;
                }
            }
            // the next item's first P is published only after these loads of O: that orders its first product
            // (which overwrites O) behind them
            tc_fence_before_sync();
            __syncwarp();
            ++item;
            if (!next(n)) break;
        }
        if (!ok && lane == 0 && *abort_flag == 0) {
            *abort_flag = 1;
            report_timeout(g.status, 0x423u);
        }
        __syncwarp();
    }

    // ---------------------------------------------------------------------- teardown
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

template <int DT, int D>
int launch_tiles(const PagedArgs &g, const deca_paged_attn_args &a, int sms, cudaStream_t st) {
    CUtensorMap tmQ, tmK, tmV;
    const uint64_t group = (uint64_t)g.group;
    {
        const uint64_t dims[4] = {(uint64_t)D, group, (uint64_t)g.Hkv, (uint64_t)g.T};
        const uint64_t strides[3] = {(uint64_t)g.q_sh * 2, (uint64_t)g.q_sh * group * 2, (uint64_t)g.q_st * 2};
        const uint32_t box[4] = {64, (uint32_t)group, 1, (uint32_t)(128 / g.group)};
        if (int rc = make_tmap_16bit(&tmQ, DT, g.q, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
    }
    if (int rc = make_cache_maps(&tmK, &tmV, DT, D, kBc, g)) return rc;
    static SmemLimitCache configured;
    if (int rc = ensure_dynamic_smem(paged_tiles_kernel<DT, D>, Layout<D>::smem, configured)) return rc;
    paged_tiles_kernel<DT, D><<<(unsigned)sms, kThreads, Layout<D>::smem, st>>>(tmQ, tmK, tmV, g);
    if (cudaError_t e = cudaGetLastError()) return (int)e;
    return launch_join<DT, D, TL>(g, (unsigned)sms, 8, st);
}

}  // namespace

size_t paged_tiles_workspace(int D, int sms) {
    return ((size_t)sms * sizeof(PartialItem) + 255) / 256 * 256 + (size_t)sms * 2 * ((size_t)TL::ROWS * D + 2 * TL::ROWS) * sizeof(float);
}

int paged_tiles_launch(const deca_paged_attn_args &a, PagedArgs &g, int sms, cudaStream_t st) {
    g.tile_tokens = 128 / g.group;
    g.meta = static_cast<PartialItem *>(a.workspace);
    g.part = reinterpret_cast<float *>(static_cast<char *>(a.workspace) + ((size_t)sms * sizeof(PartialItem) + 255) / 256 * 256);
    if (a.dtype == DECA_F16)
        return a.D == 128 ? launch_tiles<DECA_F16, 128>(g, a, sms, st) : launch_tiles<DECA_F16, 64>(g, a, sms, st);
    return a.D == 128 ? launch_tiles<DECA_BF16, 128>(g, a, sms, st) : launch_tiles<DECA_BF16, 64>(g, a, sms, st);
}

}  // namespace deca
