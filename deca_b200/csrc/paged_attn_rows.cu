// Paged attention for few query rows per request (decoding, short guesses): the cache is streamed
// once and everything else hides behind it.
//
// A CTA of four warps takes steps of 64 keys; a warp works on 16 of them by itself: it gathers its
// K and V rows through the block table into a shared-memory ring of its own with 16-byte asynchronous
// copies (no barrier between the warps), multiplies them with the 16 (or 32) packed query rows on
// mma.sync.m16n8k16, and keeps the running maximum, sum and numerators of its keys in registers.  The
// four warps are joined through shared memory at the end of an item.  With 16 rows a tcgen05 tile of 128
// rows would be idle in 7 of 8 lanes, and the tensor work is a tenth of the memory time either way:
// bytes of K and V bound this kernel.
//
// Measured (bf16, D = 128, 32 query and 8 key heads, pages of 16, device time): 64 requests of 1000 .. 8191 keys 205 us =
// 6.32 TB/s (96 % of the measured copy rate; 19 % of the tensor pipe), 100 x 1000 .. 4000 171, 16 x 2000 28.4 us, 32 x 500 .. 2500 42.6,
// 256 x 100 .. 500 67 (4.6 TB/s: the start and end of an item, 5 us, show), 1 x 8192 16.9, 1 x 333 (D = 64, 16 equal
// heads) 6.2.  A TMA producer warp ahead of four consumers gained 5 and 8 % on the first case and on the 256 requests
// but took 38 and 48 us on 16 x 2000 and 32 x 500 .. 2500 (the warps meet twice a step), and with independent consumers it was
// slower everywhere (two barrier waits a step instead of one own copy group).
//
// The running maximum moves only when a score exceeds it by 2^8 (it then rescales the numerators);
// otherwise the exponentials are taken against the old one, as in the dense attention kernels.
#include <atomic>
#include <chrono>
#include <random>

#include "paged_attn.cuh"

namespace deca {
namespace {

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <int DT>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (DT == DECA_F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// whether a packed pair holds an infinity or a NaN
template <int DT>
__device__ __forceinline__ bool pair_not_finite(uint32_t w) {
    constexpr uint32_t e = DT == DECA_F16 ? 0x7C00u : 0x7F80u;
    return (w & e) == e || ((w >> 16) & e) == e;
}

// MT tiles of 16 query rows, NW warps, ST ring slots a warp, CPS CTAs per SM.  CUT: the item list is shared out step
// by step and items are cut; else a CTA takes every gridDim.x-th (request, key head) pair whole.
template <int DT, int D, int MT, int NW, int ST, int CPS, bool CUT>
__global__ void __launch_bounds__(32 * NW, CPS) paged_rows_kernel(const PagedArgs g) {
    constexpr int ROWS = 16 * MT, kThreads = 32 * NW, kKeys = 16 * NW;
    using TL = PackedRows<ROWS, kKeys>;
    constexpr int CH = D / 8;                // 16-byte chunks per key
    constexpr uint32_t kTile = 16 * D * 2;   // one warp's K or V tile
    constexpr int KD = D / 16, ND = D / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ WorkShare share;
    __shared__ float sm[NW][ROWS], sl[NW][ROWS];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t ring = smem_u32(smem) + (uint32_t)warp * ST * 2 * kTile;
    WorkPos w;
    ReqView v;
    const int page_mask = (1 << g.page_shift) - 1;
    int part_no = 0, n_parts = 0;  // > 0: this CTA has this one part of an item
    if constexpr (CUT) {
        constexpr int kRoom = NW * ST * 2 * 16 * D * 2 / 8;
        const int found = find_part<TL>(g, w, v, part_no, n_parts);
        if (found < 0) return;
        if (found == 0) {
            n_parts = 0;
            if (!find_work<TL>(g, w, &share, reinterpret_cast<unsigned long long *>(smem), kRoom)) return;
            v = request_view(g, w.req);
        }
    } else {
        if (blockIdx.x >= (long long)g.B * g.Hkv) return;
        w.req = (int)(blockIdx.x / (unsigned)g.Hkv), w.head = (int)(blockIdx.x % (unsigned)g.Hkv), w.tile = 0, w.step = 0;
        v = request_view(g, w.req);
    }

    while (true) {
        const int steps = TL::steps(g, v, w.tile);
        const int s0 = CUT ? w.step : 0, s1 = CUT ? s0 + min(steps - s0, w.left) : steps;
        if (CUT || v.n > 0) {
            // ---- rows of this thread: lane / 4 (+ 8) of every 16
            int lim[MT][2];
            uint32_t aq[MT][KD][4];
            const int tok_first = w.tile == 0 ? 0 : (int)((unsigned long long)w.tile * ROWS / (unsigned)g.group);
            const int lim_first = min(v.shift + tok_first, v.kv - 1);
            const int kend = keys_until(v, TL::last_token(g, v, w.tile));
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    int tok, j;
                    const bool live = TL::place(g, v.n, w.tile, m * 16 + h * 8 + (lane >> 2), tok, j);
                    lim[m][h] = live ? min(v.shift + tok, v.kv - 1) : -1;
                    const char *q = g.q + 2 * (((long long)v.q0 + tok) * g.q_st + (long long)(w.head * g.group + j) * g.q_sh + 2 * (lane & 3));
#pragma unroll
                    for (int k = 0; k < KD; ++k) {
                        aq[m][k][h] = live ? *reinterpret_cast<const uint32_t *>(q + k * 32) : 0u;
                        aq[m][k][2 + h] = live ? *reinterpret_cast<const uint32_t *>(q + k * 32 + 16) : 0u;
                    }
                }
            float o[MT][ND][4], mx[MT][2], ls[MT][2];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                mx[m][0] = mx[m][1] = -INFINITY;
                ls[m][0] = ls[m][1] = 0.f;
#pragma unroll
                for (int n = 0; n < ND; ++n) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f;
            }

            // ---- the ring: tile i of the segment holds keys (s0 + i) * 64 + warp * 16 ..
            const int n_tiles = s1 - s0;
            const int *table = g.table + w.req * g.table_stride;
            auto page_of = [&](int i) {  // table entry of tile i (a tile lies within one page)
                const int key = (s0 + i) * kKeys + warp * 16;
                return i < n_tiles && key < kend ? table[key >> g.page_shift] : -1;
            };
            int pages = page_of(lane), pages_next = page_of(32 + lane);  // of 32 tiles each
            const char *kh = g.k + 2 * ((long long)(w.head * g.k_heads) * g.k_sh), *vh = g.v + 2 * ((long long)(w.head * g.v_heads) * g.v_sh);
            auto issue = [&](int i, int slot) {
                if (i < n_tiles) {
                    if ((i & 31) == 0 && i > 0) {
                        pages = pages_next;
                        pages_next = page_of(i + 32 + lane);
                    }
                    const int page = __shfl_sync(0xFFFFFFFFu, pages, i & 31);
                    const int key0 = (s0 + i) * kKeys + warp * 16;
                    const bool there = page >= 0 && page < g.num_pages;
                    const long long pg = there ? page : 0;
                    const char *kp = kh + 2 * (pg * g.k_sp), *vp = vh + 2 * (pg * g.v_sp);
                    const uint32_t dst = ring + (uint32_t)slot * 2 * kTile;
#pragma unroll
                    for (int c = 0; c < 16 * CH / 32; ++c) {
                        const int idx = c * 32 + lane, kk = idx / CH, ch = idx % CH;
                        const int row = (key0 + kk) & page_mask;
                        const bool live = there && key0 + kk < kend;
                        const uint32_t to = dst + (uint32_t)(kk * D * 2 + ((ch ^ (kk & 7)) << 4));
                        cp_async16(to, kp + 2 * ((long long)row * g.k_sr + ch * 8), live);
                        cp_async16(to + kTile, vp + 2 * ((long long)row * g.v_sr + ch * 8), live);
                    }
                }
                cp_async_commit();
            };
            __syncwarp();
#pragma unroll
            for (int i = 0; i < ST - 1; ++i) issue(i, i);
            int slot = 0, fill = ST - 1;
            for (int i = 0; i < n_tiles; ++i) {
                cp_async_wait<ST - 2>();
                __syncwarp();
                issue(i + ST - 1, fill);
                fill = fill + 1 == ST ? 0 : fill + 1;
                const uint32_t tk = ring + (uint32_t)slot * 2 * kTile, tv = tk + kTile;
                slot = slot + 1 == ST ? 0 : slot + 1;
                const int key0 = (s0 + i) * kKeys + warp * 16;
                if (key0 >= kend) continue;

                // S = Q K^T
                float s[MT][2][4];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int n = 0; n < 2; ++n) s[m][n][0] = s[m][n][1] = s[m][n][2] = s[m][n][3] = 0.f;
                const int quad = lane >> 3, l8 = lane & 7;
#pragma unroll
                for (int k = 0; k < KD; ++k) {
                    uint32_t b[4];
                    const int kk = (quad >> 1) * 8 + l8, ch = k * 2 + (quad & 1);
                    ldsm4(b, tk + (uint32_t)(kk * D * 2 + ((ch ^ l8) << 4)));
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        mma16816<DT>(s[m][0], aq[m][k], b[0], b[1]);
                        mma16816<DT>(s[m][1], aq[m][k], b[2], b[3]);
                    }
                }
                // scores to the exponent's domain, masked where the row does not see the key
                const bool masked = key0 + 15 > lim_first;
                bool raise = false;
                float top[MT][2];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    top[m][0] = top[m][1] = -INFINITY;
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float x = s[m][n][e] * g.sl2;
                            if (masked && key0 + n * 8 + 2 * (lane & 3) + (e & 1) > lim[m][e >> 1]) x = -INFINITY;
                            s[m][n][e] = x;
                            top[m][e >> 1] = fmaxf(top[m][e >> 1], x);
                        }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        top[m][h] = fmaxf(top[m][h], __shfl_xor_sync(0xFFFFFFFFu, top[m][h], 1));
                        top[m][h] = fmaxf(top[m][h], __shfl_xor_sync(0xFFFFFFFFu, top[m][h], 2));
                        raise = raise || top[m][h] > mx[m][h] + 8.0f;
                    }
                }
                if (__any_sync(0xFFFFFFFFu, raise)) {
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        float f[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float up = fmaxf(mx[m][h], top[m][h]);
                            f[h] = mx[m][h] == -INFINITY ? 0.f : exp2f(mx[m][h] - up);
                            mx[m][h] = up;
                            ls[m][h] *= f[h];
                        }
#pragma unroll
                        for (int n = 0; n < ND; ++n) {
                            o[m][n][0] *= f[0], o[m][n][1] *= f[0];
                            o[m][n][2] *= f[1], o[m][n][3] *= f[1];
                        }
                    }
                }
                uint32_t p[MT][4];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float base = mx[m][h] == -INFINITY ? 0.f : mx[m][h];
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            const float e0 = ex2_approx(s[m][n][2 * h] - base), e1 = ex2_approx(s[m][n][2 * h + 1] - base);
                            ls[m][h] += e0 + e1;
                            s[m][n][2 * h] = e0, s[m][n][2 * h + 1] = e1;
                            p[m][2 * n + h] = Pack16<DT>::pack(e0, e1);  // rounded for the product; the sum is not
                        }
                    }
                }
                // A key that only some rows see may hold anything: 0 * inf would reach the others
                bool bad = false;
                if (masked) {
                    for (int c = 0; c < 16 * CH / 32; ++c) {
                        const int idx = c * 32 + lane, kk = idx / CH, ch = idx % CH;
                        if (key0 + kk <= lim_first) continue;
                        uint32_t x[4];
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                     : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                                     : "r"(tv + (uint32_t)(kk * D * 2 + (ch << 4)))
                                     : "memory");
                        bad = bad || pair_not_finite<DT>(x[0]) || pair_not_finite<DT>(x[1]) || pair_not_finite<DT>(x[2]) ||
                              pair_not_finite<DT>(x[3]);
                    }
                    bad = __any_sync(0xFFFFFFFFu, bad) != 0;
                }
                if (!bad) {
                    // O += P V
#pragma unroll
                    for (int n = 0; n < D / 16; ++n) {
                        uint32_t b[4];
                        const int kk = (quad & 1) * 8 + l8, ch = n * 2 + (quad >> 1);
                        ldsm4_trans(b, tv + (uint32_t)(kk * D * 2 + ((ch ^ l8) << 4)));
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            mma16816<DT>(o[m][2 * n], p[m], b[0], b[1]);
                            mma16816<DT>(o[m][2 * n + 1], p[m], b[2], b[3]);
                        }
                    }
                } else {
                    // the same product key by key, leaving out what a row does not see
#pragma unroll
                    for (int kk = 0; kk < 16; ++kk) {
                        const int src = (lane & ~3) | ((kk & 7) >> 1);
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            const float p0 = __shfl_sync(0xFFFFFFFFu, s[m][kk >> 3][kk & 1], src);
                            const float p1 = __shfl_sync(0xFFFFFFFFu, s[m][kk >> 3][2 + (kk & 1)], src);
                            const bool see0 = key0 + kk <= lim[m][0], see1 = key0 + kk <= lim[m][1];
#pragma unroll
                            for (int n = 0; n < ND; ++n) {
                                uint32_t x;
                                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(tv + (uint32_t)(kk * D * 2 + ((n ^ (kk & 7)) << 4) + 4 * (lane & 3))) : "memory");
                                const float2 f = Pack16<DT>::unpack(x);
                                if (see0) o[m][n][0] = fmaf(p0, f.x, o[m][n][0]), o[m][n][1] = fmaf(p0, f.y, o[m][n][1]);
                                if (see1) o[m][n][2] = fmaf(p1, f.x, o[m][n][2]), o[m][n][3] = fmaf(p1, f.y, o[m][n][3]);
                            }
                        }
                    }
                }
            }
            cp_async_wait<0>();
            __syncwarp();

            // ---- join the four warps: numerators into each warp's ring (swizzled by 32 bytes), statistics beside
            float *mine = reinterpret_cast<float *>(smem + (size_t)warp * ST * 2 * kTile);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = m * 16 + h * 8 + (lane >> 2);
                    float l = ls[m][h];
                    l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
                    l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
                    if ((lane & 3) == 0) sm[warp][row] = mx[m][h], sl[warp][row] = l;
#pragma unroll
                    for (int n = 0; n < ND; ++n)
                        *reinterpret_cast<float2 *>(mine + row * D + ((n ^ (row & 7)) * 8) + 2 * (lane & 3)) =
                            make_float2(o[m][n][2 * h], o[m][n][2 * h + 1]);
                }
            __syncthreads();
            constexpr int kPerRow = kThreads / ROWS;  // threads that share a row
            const int row = tid / kPerRow;
            float topw = -INFINITY;
#pragma unroll
            for (int i = 0; i < NW; ++i) topw = fmaxf(topw, sm[i][row]);
            const float base = topw == -INFINITY ? 0.f : topw;
            float wt[NW], l = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                wt[i] = exp2f(sm[i][row] - base);
                l = fmaf(wt[i], sl[i][row], l);
            }
            const bool whole_item = !CUT || (s0 == 0 && s1 == steps);
            const bool starts = s0 == 0;
            float *part = g.part + ((size_t)blockIdx.x * 2 + (starts ? 1 : 0)) * kPartFloats<ROWS, D>;
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            int tok, j;
            const bool live = TL::place(g, v.n, w.tile, row, tok, j);
            char *out = g.o + 2 * (((long long)v.q0 + tok) * g.o_st + (long long)(w.head * g.group + j) * g.o_sh);
#pragma unroll
            for (int n0 = 0; n0 < ND; n0 += kPerRow) {
                const int n = n0 + tid % kPerRow;
                if (n >= ND) break;
                float acc[8] = {};
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    const float *src = reinterpret_cast<const float *>(smem + (size_t)i * ST * 2 * kTile) + row * D + ((n ^ (row & 7)) * 8);
                    const float4 x = *reinterpret_cast<const float4 *>(src), y = *reinterpret_cast<const float4 *>(src + 4);
                    acc[0] = fmaf(wt[i], x.x, acc[0]), acc[1] = fmaf(wt[i], x.y, acc[1]);
                    acc[2] = fmaf(wt[i], x.z, acc[2]), acc[3] = fmaf(wt[i], x.w, acc[3]);
                    acc[4] = fmaf(wt[i], y.x, acc[4]), acc[5] = fmaf(wt[i], y.y, acc[5]);
                    acc[6] = fmaf(wt[i], y.z, acc[6]), acc[7] = fmaf(wt[i], y.w, acc[7]);
                }
                if (whole_item) {
                    if (live)
                        *reinterpret_cast<uint4 *>(out + n * 16) =
                            make_uint4(Pack16<DT>::pack(acc[0] * inv, acc[1] * inv), Pack16<DT>::pack(acc[2] * inv, acc[3] * inv),
                                       Pack16<DT>::pack(acc[4] * inv, acc[5] * inv), Pack16<DT>::pack(acc[6] * inv, acc[7] * inv));
                } else {
                    float4 *dst = reinterpret_cast<float4 *>(part + (size_t)row * D + n * 8);
                    dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
                    dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
                }
            }
            if constexpr (CUT) {
                if (!whole_item) {
                    if (tid % kPerRow == 0) part[(size_t)ROWS * D + row] = topw, part[(size_t)ROWS * D + ROWS + row] = l;
                    // Tell the others, and see whether they have all told: the last one to tell (or two that tell at
                    // the same time, with the same result) joins.  The flags hold a number of this launch and are
                    // cleared by whoever joins, so what the workspace held before, or a replay of the same captured
                    // launch, is not taken for it.
                    __shared__ int all;
                    __syncthreads();
                    int c0 = (int)blockIdx.x - part_no, n = n_parts;
                    if (n_parts == 0) {
                        const long long item = share.end - w.left - s0;  // its first step in the list
                        c0 = cta_of(&share, item), n = cta_of(&share, item + steps - 1) - c0 + 1;
                    }
                    auto flag = [&](int i) { return g.flags + (size_t)(c0 + i) * 2 + (i == 0 ? 1 : 0); };
                    if (warp == 0) {
                        if (lane == 0) {
                            __threadfence();
                            *reinterpret_cast<volatile unsigned long long *>(g.flags + (size_t)blockIdx.x * 2 + (starts ? 1 : 0)) = g.tag;
                            __threadfence();
                        }
                        __syncwarp();
                        bool there = true;
                        for (int i = lane; i < n; i += 32) there = there && *reinterpret_cast<volatile unsigned long long *>(flag(i)) == g.tag;
                        there = __all_sync(0xFFFFFFFFu, there) != 0;
                        __threadfence();
                        if (lane == 0) all = there ? 1 : 0;
                    }
                    __syncthreads();
                    if (all) {
                        auto part_of = [&](int i) { return g.part + ((size_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * kPartFloats<ROWS, D>; };
                        for (int r = warp; r < ROWS; r += NW) {
                            int t, jj;
                            if (!TL::place(g, v.n, w.tile, r, t, jj)) break;
                            float acc[D / 32], sum;
                            join_row<ROWS, D, 16>(part_of, n, r, lane, acc, sum);
                            store_joined<DT, D>(g.o + 2 * (((long long)v.q0 + t) * g.o_st + (long long)(w.head * g.group + jj) * g.o_sh), lane, acc, sum);
                        }
                        for (int i = tid; i < n; i += kThreads) *reinterpret_cast<volatile unsigned long long *>(flag(i)) = 0ull;
                    }
                }
            }
            __syncthreads();  // the rings and statistics are free again
        }
        if constexpr (CUT) {
            w.left -= s1 - s0;
            if (w.left <= 0 || n_parts > 0 || !next_item<TL>(g, w, v)) break;
        } else if (++w.tile >= TL::tiles(g, v)) {
            w.tile = 0;
            const long long pair = (long long)w.req * g.Hkv + w.head + gridDim.x;
            if (pair >= (long long)g.B * g.Hkv) break;
            w.req = (int)(pair / g.Hkv), w.head = (int)(pair % g.Hkv);
            v = request_view(g, w.req);
        }
    }
}

template <int DT, int D, int MT, int NW, int ST, int CPS, bool CUT>
int launch_cfg(const PagedArgs &g, int sms, cudaStream_t st) {
    constexpr size_t smem = (size_t)NW * ST * 2 * 16 * D * 2;
    static SmemLimitCache configured;
    if (int rc = ensure_dynamic_smem(paged_rows_kernel<DT, D, MT, NW, ST, CPS, CUT>, smem, configured)) return rc;
    long long ctas = (long long)CPS * sms;
    if (!CUT && (long long)g.B * g.Hkv < ctas) ctas = (long long)g.B * g.Hkv;
    paged_rows_kernel<DT, D, MT, NW, ST, CPS, CUT><<<(unsigned)ctas, 32 * NW, smem, st>>>(g);
    return (int)cudaGetLastError();
}
// Four warps; three ring slots of 16 keys each, and as many CTAs as fit: two (D = 128, or 32 rows, by registers) or
// four an SM.  Two-warp CTAs (more of them) were slower wherever items are cut: twice the parts to join.
template <int D, int MT>
constexpr int kCtasPerSm = D == 64 && MT == 1 ? 4 : 2;

template <int DT, int D, int MT>
int launch_rows(const PagedArgs &g, bool cut, int sms, cudaStream_t st) {
    return cut ? launch_cfg<DT, D, MT, 4, 3, kCtasPerSm<D, MT>, true>(g, sms, st)
               : launch_cfg<DT, D, MT, 4, 3, kCtasPerSm<D, MT>, false>(g, sms, st);
}

template <int DT>
int launch_rows_dtype(const PagedArgs &g, int D, int mt, bool cut, int sms, cudaStream_t st) {
    if (D == 128) return mt == 1 ? launch_rows<DT, 128, 1>(g, cut, sms, st) : launch_rows<DT, 128, 2>(g, cut, sms, st);
    return mt == 1 ? launch_rows<DT, 64, 1>(g, cut, sms, st) : launch_rows<DT, 64, 2>(g, cut, sms, st);
}

size_t flag_bytes(int ctas) { return ((size_t)ctas * 2 * sizeof(unsigned long long) + 255) / 256 * 256; }

// A number that no other launch of any process carries, but for one chance in 2^64 or so.
unsigned long long launch_tag() {
    static std::atomic<unsigned long long> next{[] {
        unsigned long long seed = (unsigned long long)std::chrono::system_clock::now().time_since_epoch().count();
        try {
            std::random_device rd;
            seed ^= ((unsigned long long)rd() << 32) ^ (unsigned long long)rd();
        } catch (...) {  // no source of randomness: the clock and where the library lies have to do
            seed ^= (unsigned long long)reinterpret_cast<uintptr_t>(&flag_bytes) << 20;
        }
        return seed;
    }()};
    unsigned long long t = next.fetch_add(0x9E3779B97F4A7C15ull);  // odd: runs through all 2^64 values
    return t ? t : next.fetch_add(0x9E3779B97F4A7C15ull);          // 0 is a cleared flag
}

}  // namespace

int paged_rows_ctas(int D, int mt, int sms) { return (D == 64 && mt == 1 ? kCtasPerSm<64, 1> : kCtasPerSm<128, 1>) * sms; }

// bytes of workspace for `mt` tiles of 16 rows where items are cut: two flags and two partial results per CTA
size_t paged_rows_workspace(int D, int mt, int sms) {
    const size_t rows = 16 * (size_t)mt, ctas = (size_t)paged_rows_ctas(D, mt, sms);
    return flag_bytes((int)ctas) + ctas * 2 * (rows * D + 2 * rows) * sizeof(float);
}

int paged_rows_launch(const deca_paged_attn_args &a, PagedArgs &g, int mt, bool cut, int sms, cudaStream_t st) {
    g.flags = static_cast<unsigned long long *>(a.workspace);
    g.part = reinterpret_cast<float *>(static_cast<char *>(a.workspace) + flag_bytes(paged_rows_ctas(a.D, mt, sms)));
    g.max_parts = 32;
    g.min_steps = 4;
    if (cut) g.tag = launch_tag();
    return a.dtype == DECA_F16 ? launch_rows_dtype<DECA_F16>(g, a.D, mt, cut, sms, st)
                               : launch_rows_dtype<DECA_BF16>(g, a.D, mt, cut, sms, st);
}

}  // namespace deca
