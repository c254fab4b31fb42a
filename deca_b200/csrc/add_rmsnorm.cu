// Residual addition + RMSNorm with a 16-bit or an e4m3 output (deca_add_rmsnorm).
//
//   h = x + res;  y = h * rsqrt(sum h^2 / N + eps) * w;  out dt(h) and dt(y), or e4m3(y / s) with
//   s = max |y| / 448 over the row or a group of columns.
//
// One pass: a row's h stays in fp32 registers between the sum of squares and the output, so every element
// is read once and written once, which is the floor of an HBM-bound operator: 8 bytes per element, 7
// with the 8-bit output.  A warp takes spans of 256 columns, eight per lane, in accesses of V elements: V =
// 8 (16 bytes) where rows are aligned, else 4, 2 or 1, with the lanes of one access side by side, so that
// an odd row length costs instructions but not sectors.  The columns of a scale group (32 .. 256) then lie
// in one warp's span and its maximum takes shuffles alone.
// Rows beyond the registers of a CTA are streamed twice (three times for one scale a row).
//
// Bound by HBM (measured copy rate 6.57 TB/s).  bf16, device time: 16384 x 4096 to 16 bits 81.0 us = 6.63 TB/s,
// 8000 x 12000 117.8 us = 6.52; to e4m3 16384 x 8192 per row 155.5 us = 6.04 TB/s, per 128 columns 165.3 us = 5.71
// (issue slots 78 % busy: the conversions and maxima show), 1021 x 5000 per row 9.2 us; rows of 1001 elements (2-byte
// accesses) 3.25 TB/s, 19.7 us at 8000 x 1001 (16-byte accesses shifted through shared memory: 23.2).  16 x 4096: 2.3 us,
// launch latency; there a warp takes one span instead of two (256 x 8192 3.9 us), which is what shortens the chain of
// loads.
#include "common.cuh"
#include "overlap.cuh"
#include "ptx.cuh"

namespace deca {
namespace {

constexpr int kMaxRegThreads = 512;
constexpr int kGrouped = 2;  // DECA_OUT_E4M3 with a scale per group of columns
constexpr float kE4m3Max = 448.0f;
constexpr float kMinScale = 1.17549435e-38f;  // below it 1 / s is no finite number: the group is written as zeros

struct AddNormArgs {
    const char *x, *r, *w;
    char *h, *y;
    float *scales;
    long long M;
    long long sx, sr, sh, sy;  // row strides in elements
    int N;
    int tpr;  // threads per row
    int group_shift, n_groups;  // log2 of a scale group's columns (0: one scale a row)
    float eps, inv_n;
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Two fp32 operations in one instruction (the 8-bit forms issue in 78 % of the cycles without them).
__device__ __forceinline__ void add_pairs(float (&a)[8], const float (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) f32x2_unpack(f32x2_add(f32x2_pack(a[i], a[i + 1]), f32x2_pack(b[i], b[i + 1])), a[i], a[i + 1]);
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// y = h * rs * w
__device__ __forceinline__ void scale_pairs(float (&h)[8], float rs, const float (&w)[8]) {
    const uint64_t r2 = f32x2_pack(rs, rs);
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        f32x2_unpack(mul_pair(mul_pair(f32x2_pack(h[i], h[i + 1]), r2), f32x2_pack(w[i], w[i + 1])), h[i], h[i + 1]);
}
__device__ __forceinline__ uint64_t square_pairs(const float (&h)[8], uint64_t sum) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint64_t p = f32x2_pack(h[i], h[i + 1]);
        sum = f32x2_fma(p, p, sum);
    }
    return sum;
}
__device__ __forceinline__ float max3_nan_abs(float m, float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}

template <int DT>
__device__ __forceinline__ float load1(const char *p) {
    if constexpr (DT == DECA_F16) return __half2float(*reinterpret_cast<const __half *>(p));
    return __bfloat162float(*reinterpret_cast<const __nv_bfloat16 *>(p));
}
template <int DT>
__device__ __forceinline__ void store1(char *p, float v) {
    if constexpr (DT == DECA_F16)
        *reinterpret_cast<__half *>(p) = __float2half_rn(v);
    else
        *reinterpret_cast<__nv_bfloat16 *>(p) = __float2bfloat16_rn(v);
}

// Column of element i (0 .. 7) of a lane in the span that starts at `span`: access i / V, V elements each.
template <int V>
__device__ __forceinline__ int column(int span, int lane, int i) {
    return span + (i / V) * 32 * V + lane * V + i % V;
}

// A lane's eight elements of a span as fp32, zeros behind the row's end (N is a multiple of V).
template <int DT, int V, bool STREAM>
__device__ __forceinline__ void load8(float (&f)[8], const char *row, int span, int lane, int N) {
#pragma unroll
    for (int a = 0; a < 8; a += V) {
        const int col = column<V>(span, lane, a);
        const char *p = row + (size_t)col * 2;
        if constexpr (V == 1) {
            f[a] = col < N ? load1<DT>(p) : 0.f;
        } else {
            uint32_t d[V / 2];
#pragma unroll
            for (int k = 0; k < V / 2; ++k) d[k] = 0u;
            if (col < N) {
                if constexpr (V == 8 && STREAM)
                    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                                 : "l"(p));
                else if constexpr (V == 8)
                    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "l"(p));
                else if constexpr (V == 4)
                    asm volatile("ld.global.v2.u32 {%0,%1}, [%2];" : "=r"(d[0]), "=r"(d[1]) : "l"(p));
                else
                    asm volatile("ld.global.u32 %0, [%1];" : "=r"(d[0]) : "l"(p));
            }
#pragma unroll
            for (int k = 0; k < V / 2; ++k) {
                const float2 v = Pack16<DT>::unpack(d[k]);
                f[a + 2 * k] = v.x, f[a + 2 * k + 1] = v.y;
            }
        }
    }
}

template <int DT, int V>
__device__ __forceinline__ void store8(char *row, int span, int lane, int N, const float (&f)[8]) {
#pragma unroll
    for (int a = 0; a < 8; a += V) {
        const int col = column<V>(span, lane, a);
        char *p = row + (size_t)col * 2;
        if (col >= N) continue;
        if constexpr (V == 1) {
            store1<DT>(p, f[a]);
        } else if constexpr (V == 8) {
            asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(Pack16<DT>::pack(f[0], f[1])),
                         "r"(Pack16<DT>::pack(f[2], f[3])), "r"(Pack16<DT>::pack(f[4], f[5])), "r"(Pack16<DT>::pack(f[6], f[7]))
                         : "memory");
        } else if constexpr (V == 4) {
            *reinterpret_cast<uint2 *>(p) = make_uint2(Pack16<DT>::pack(f[a], f[a + 1]), Pack16<DT>::pack(f[a + 2], f[a + 3]));
        } else {
            *reinterpret_cast<uint32_t *>(p) = Pack16<DT>::pack(f[a], f[a + 1]);
        }
    }
}

// Two values to e4m3 (round to nearest even, saturating, NaN kept), the first in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t v;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(v) : "f"(hi), "f"(lo));
    return v;
}

template <int V>
__device__ __forceinline__ void store_e4m3(char *row, int span, int lane, int N, const float (&y)[8], const float (&inv)[8 / V]) {
#pragma unroll
    for (int a = 0; a < 8; a += V) {
        const int col = column<V>(span, lane, a);
        const float s = inv[a / V];
        if (col >= N) continue;
        if constexpr (V == 8)
            asm volatile("st.global.cs.v2.u32 [%0], {%1,%2};" ::"l"(row + col),
                         "r"(e4m3x2(y[0] * s, y[1] * s) | (e4m3x2(y[2] * s, y[3] * s) << 16)),
                         "r"(e4m3x2(y[4] * s, y[5] * s) | (e4m3x2(y[6] * s, y[7] * s) << 16))
                         : "memory");
        else if constexpr (V == 4)
            *reinterpret_cast<uint32_t *>(row + col) =
                e4m3x2(y[a] * s, y[a + 1] * s) | (e4m3x2(y[a + 2] * s, y[a + 3] * s) << 16);
        else if constexpr (V == 2)
            *reinterpret_cast<uint16_t *>(row + col) = (uint16_t)e4m3x2(y[a] * s, y[a + 1] * s);
        else
            row[col] = (char)(e4m3x2(y[a] * s, 0.f) & 0xFFu);
    }
}

__device__ __forceinline__ float abs_max8(const float (&y)[8]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) m = max3_nan_abs(m, y[i], y[i + 1]);
    return m;
}

// Scale and its inverse of a group whose largest |y| is `m`.
__device__ __forceinline__ void scale_of(float m, float &s, float &inv) {
    s = m * (1.0f / kE4m3Max);
    inv = s >= kMinScale ? __frcp_rn(s) : 0.f;
}

// A span of a grouped e4m3 output: maxima over the lanes (and accesses) that share a group, scales, store.
// Called by all lanes of a warp, with y = 0 behind the row's end.
template <int V>
__device__ __forceinline__ void store_grouped(const AddNormArgs &a, long long row, char *yrow, int span, int lane, const float (&y)[8]) {
    constexpr int A = 8 / V;  // accesses
    float m[A], inv[A];
#pragma unroll
    for (int k = 0; k < A; ++k) {
        m[k] = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) m[k] = max_nan(m[k], fabsf(y[k * V + i]));
    }
    const int group = 1 << a.group_shift;
    // groups wider than an access of the warp (32 V columns): neighbouring accesses share a maximum
#pragma unroll
    for (int w = 1; w < A; w *= 2)
        if (group >= 64 * V * w) {
#pragma unroll
            for (int k = 0; k < A; k += 2 * w) {
                float t = max_nan(m[k], m[k + w]);
#pragma unroll
                for (int i = 0; i < 2 * w; ++i) m[k + i] = t;
            }
        }
    const int lanes = min(group / V, 32);
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1)
        if (s < lanes) {
#pragma unroll
            for (int k = 0; k < A; ++k) m[k] = max_nan(m[k], __shfl_xor_sync(0xFFFFFFFFu, m[k], s));
        }
#pragma unroll
    for (int k = 0; k < A; ++k) {
        float scale;
        scale_of(m[k], scale, inv[k]);
        const int col = column<V>(span, lane, k * V);
        if ((col & (group - 1)) == 0 && col < a.N) a.scales[row * a.n_groups + (col >> a.group_shift)] = scale;
    }
    store_e4m3<V>(yrow, span, lane, a.N, y, inv);
}

template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, float *red, int nw, int row_warp0, int wr, int lane) {
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) {
        const float o = __shfl_xor_sync(0xFFFFFFFFu, v, s);
        v = MAX ? max_nan(v, o) : v + o;
    }
    if (nw > 1) {
        if (lane == 0) red[row_warp0 + wr] = v;
        __syncthreads();
        v = red[row_warp0];
        for (int i = 1; i < nw; ++i) v = MAX ? max_nan(v, red[row_warp0 + i]) : v + red[row_warp0 + i];
    }
    return v;
}

// The row in registers: C spans per warp, `rpb` rows per CTA.  OUT: DECA_OUT_SAME, DECA_OUT_E4M3 (one scale a
// row) or kGrouped.
template <int DT, int OUT, int C, int V>
__global__ void __launch_bounds__(kMaxRegThreads) add_rmsnorm_reg_kernel(const AddNormArgs a) {
    __shared__ float red[2][32];
    const int t = threadIdx.x % a.tpr, rb = threadIdx.x / a.tpr;
    const int lane = threadIdx.x & 31, wr = t >> 5, nw = a.tpr >> 5;
    const long long row = (long long)blockIdx.x * (blockDim.x / a.tpr) + rb;
    const bool live = row < a.M;  // the threads of a row behind the last one take part in the barriers only
    const int N = live ? a.N : 0;
    const char *xrow = a.x + row * a.sx * 2, *rrow = a.r + row * a.sr * 2;
    char *hrow = a.h + row * a.sh * 2, *yrow = a.y + row * a.sy * (OUT == DECA_OUT_SAME ? 2 : 1);

    // fp32 pairs pay with one scale a row (16384 x 8192: 161 -> 156 us); with grouped scales they cost (165 -> 194), and
    // the 16-bit output is at the memory's rate either way
    constexpr bool kPairs = OUT == DECA_OUT_E4M3;
    float h[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int span = (c * nw + wr) * 256;
        float r[8];
        load8<DT, V, true>(h[c], xrow, span, lane, N);
        load8<DT, V, true>(r, rrow, span, lane, N);
        if constexpr (kPairs) {
            add_pairs(h[c], r);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] += r[i];
        }
    }
    float ss = 0.f;
    if constexpr (kPairs) {
        uint64_t squares = 0ull;
#pragma unroll
        for (int c = 0; c < C; ++c) squares = square_pairs(h[c], squares);
        float odd;
        f32x2_unpack(squares, ss, odd);
        ss += odd;
    } else {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(h[c][i], h[c][i], ss);
    }
    ss = row_reduce<false>(ss, red[0], nw, rb * nw, wr, lane);
    const float rs = rsqrtf(fmaf(ss, a.inv_n, a.eps));

    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int span = (c * nw + wr) * 256;
        store8<DT, V>(hrow, span, lane, N, h[c]);
        float w[8];
        load8<DT, V, false>(w, a.w, span, lane, N);
        if constexpr (kPairs) {
            scale_pairs(h[c], rs, w);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = h[c][i] * rs * w[i];
        }
        if constexpr (OUT == DECA_OUT_SAME)
            store8<DT, V>(yrow, span, lane, N, h[c]);
        else if constexpr (OUT == DECA_OUT_E4M3)
            amax = max_nan(amax, abs_max8(h[c]));
        else if (live && span < N)
            store_grouped<V>(a, row, yrow, span, lane, h[c]);
    }
    if constexpr (OUT == DECA_OUT_E4M3) {
        amax = row_reduce<true>(amax, red[1], nw, rb * nw, wr, lane);
        float scale, inv1, inv[8 / V];
        scale_of(amax, scale, inv1);
#pragma unroll
        for (int k = 0; k < 8 / V; ++k) inv[k] = inv1;
        if (live && t == 0) a.scales[row] = scale;
#pragma unroll
        for (int c = 0; c < C; ++c) store_e4m3<V>(yrow, (c * nw + wr) * 256, lane, N, h[c], inv);
    }
}

// Rows of any length: the row is read once for the sum of squares, (one scale a row) once for the
// maximum and once for the output; re-reads come from L2.
template <int DT, int OUT, int V>
__global__ void __launch_bounds__(kMaxRegThreads) add_rmsnorm_stream_kernel(const AddNormArgs a) {
    __shared__ float red[2][32];
    const int t = threadIdx.x, lane = t & 31, wr = t >> 5, nw = blockDim.x >> 5;
    const long long row = blockIdx.x;
    const char *xrow = a.x + row * a.sx * 2, *rrow = a.r + row * a.sr * 2;
    char *hrow = a.h + row * a.sh * 2, *yrow = a.y + row * a.sy * (OUT == DECA_OUT_SAME ? 2 : 1);
    const int step = nw * 256, first = wr * 256;
    auto load_h = [&](float (&h)[8], int span) {
        float r[8];
        load8<DT, V, false>(h, xrow, span, lane, a.N);
        load8<DT, V, false>(r, rrow, span, lane, a.N);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] += r[i];
    };
    auto scale_h = [&](float (&y)[8], int span, float rs) {
        float w[8];
        load8<DT, V, false>(w, a.w, span, lane, a.N);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * rs * w[i];
    };
    float ss = 0.f;
    for (int span = first; span < a.N; span += step) {
        float h[8];
        load_h(h, span);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(h[i], h[i], ss);
    }
    ss = row_reduce<false>(ss, red[0], nw, 0, wr, lane);
    const float rs = rsqrtf(fmaf(ss, a.inv_n, a.eps));
    float inv[8 / V];
    if constexpr (OUT == DECA_OUT_E4M3) {
        float amax = 0.f;
        for (int span = first; span < a.N; span += step) {
            float y[8];
            load_h(y, span);
            scale_h(y, span, rs);
            amax = max_nan(amax, abs_max8(y));
        }
        amax = row_reduce<true>(amax, red[1], nw, 0, wr, lane);
        float scale, inv1;
        scale_of(amax, scale, inv1);
#pragma unroll
        for (int k = 0; k < 8 / V; ++k) inv[k] = inv1;
        if (t == 0) a.scales[row] = scale;
    }
    // every element is read again and then written by the same thread, so H may be X or R
    for (int span = first; span < a.N; span += step) {
        float y[8];
        load_h(y, span);
        store8<DT, V>(hrow, span, lane, a.N, y);
        scale_h(y, span, rs);
        if constexpr (OUT == DECA_OUT_SAME)
            store8<DT, V>(yrow, span, lane, a.N, y);
        else if constexpr (OUT == DECA_OUT_E4M3)
            store_e4m3<V>(yrow, span, lane, a.N, y, inv);
        else
            store_grouped<V>(a, row, yrow, span, lane, y);
    }
}

template <int DT, int OUT, int V>
int launch(const AddNormArgs &a, int spans, int rpb, cudaStream_t st) {
    if (spans == 0) {
        if (a.M > 2147483647ll) return DECA_ERR_SHAPE;
        add_rmsnorm_stream_kernel<DT, OUT, V><<<(unsigned)a.M, 512, 0, st>>>(a);
        return (int)cudaGetLastError();
    }
    const long long grid = (a.M + rpb - 1) / rpb;
    if (grid > 2147483647ll) return DECA_ERR_SHAPE;
    const unsigned g = (unsigned)grid, threads = (unsigned)(a.tpr * rpb);
    switch (spans) {
        case 1: add_rmsnorm_reg_kernel<DT, OUT, 1, V><<<g, threads, 0, st>>>(a); break;
        case 2: add_rmsnorm_reg_kernel<DT, OUT, 2, V><<<g, threads, 0, st>>>(a); break;
        case 3: add_rmsnorm_reg_kernel<DT, OUT, 3, V><<<g, threads, 0, st>>>(a); break;
        case 4: add_rmsnorm_reg_kernel<DT, OUT, 4, V><<<g, threads, 0, st>>>(a); break;
        default: add_rmsnorm_reg_kernel<DT, OUT, 8, V><<<g, threads, 0, st>>>(a); break;
    }
    return (int)cudaGetLastError();
}

template <int DT, int OUT>
int launch_width(const AddNormArgs &a, int v, int spans, int rpb, cudaStream_t st) {
    switch (v) {
        case 8: return launch<DT, OUT, 8>(a, spans, rpb, st);
        case 4: return launch<DT, OUT, 4>(a, spans, rpb, st);
        case 2: return launch<DT, OUT, 2>(a, spans, rpb, st);
        default: return launch<DT, OUT, 1>(a, spans, rpb, st);
    }
}

template <int DT>
int launch_out(const AddNormArgs &a, int out, int v, int spans, int rpb, cudaStream_t st) {
    if (out == DECA_OUT_SAME) return launch_width<DT, DECA_OUT_SAME>(a, v, spans, rpb, st);
    return a.group_shift > 0 ? launch_width<DT, kGrouped>(a, v, spans, rpb, st)
                             : launch_width<DT, DECA_OUT_E4M3>(a, v, spans, rpb, st);
}

}  // namespace
}  // namespace deca

using namespace deca;

extern "C" int deca_add_rmsnorm(int dtype, const void *X, int64_t x_stride, const void *R, int64_t r_stride,
                                const void *W, void *H, int64_t h_stride, void *Y, int64_t y_stride, float *scales,
                                int64_t M, int64_t N, float eps, int out, int group, void *stream) {
    if (dtype != DECA_F16 && dtype != DECA_BF16) return DECA_ERR_UNSUPPORTED;
    if (out != DECA_OUT_SAME && out != DECA_OUT_E4M3) return DECA_ERR_UNSUPPORTED;
    if (M < 0 || N <= 0 || N > (1ll << 30)) return DECA_ERR_SHAPE;
    if (out == DECA_OUT_SAME ? group != 0 : (group != 0 && group != 32 && group != 64 && group != 128 && group != 256))
        return DECA_ERR_CONFIG;
    if (M == 0) return DECA_OK;
    if (!X || !R || !W || !H || !Y || (out == DECA_OUT_E4M3 && !scales)) return DECA_ERR_NULL;
    if (M > 1 && (x_stride < N || r_stride < N || h_stride < N || y_stride < N)) return DECA_ERR_SHAPE;
    const int out_bytes = out == DECA_OUT_SAME ? 2 : 1;
    if (!aligned_to(X, 2) || !aligned_to(R, 2) || !aligned_to(W, 2) || !aligned_to(H, 2) || !aligned_to(Y, out_bytes) ||
        !aligned_to(scales, 4))
        return DECA_ERR_ALIGN;
    // Every element is read and written by one thread, which has read it from X and R before it writes H and Y: H and Y may
    // each replace one of them.  W and the scales are shared between threads.
    {
        const Region x = region(X, 2 * N, M, 2 * x_stride), r = region(R, 2 * N, M, 2 * r_stride), w = region(W, 2 * N);
        const Region h = region(H, 2 * N, M, 2 * h_stride), y = region(Y, out_bytes * N, M, out_bytes * y_stride);
        const Region s = region(scales, 4, out == DECA_OUT_E4M3 ? M * (group ? (N + group - 1) / group : 1) : 0, 4);
        for (const Region &in : {x, r}) {
            if (!regions_equal(h, in) && !regions_apart(h, in)) return DECA_ERR_UNSUPPORTED;
            if (!regions_equal(y, in) && !regions_apart(y, in)) return DECA_ERR_UNSUPPORTED;
        }
        if (!regions_apart(h, y) || !regions_apart(h, w) || !regions_apart(y, w)) return DECA_ERR_UNSUPPORTED;
        for (const Region &other : {x, r, w, h, y})
            if (!regions_apart(s, other)) return DECA_ERR_UNSUPPORTED;
    }
    // elements per access: the widest that the row length, the strides and the bases allow
    int v = 8;
    auto fits = [&](int w) {
        const bool strides = M == 1 || (x_stride % w == 0 && r_stride % w == 0 && h_stride % w == 0 && y_stride % w == 0);
        return N % w == 0 && strides && aligned_to(X, 2 * w) && aligned_to(R, 2 * w) && aligned_to(W, 2 * w) &&
               aligned_to(H, 2 * w) && aligned_to(Y, w * out_bytes);
    };
    while (v > 1 && !fits(v)) v /= 2;
    AddNormArgs a;
    a.x = static_cast<const char *>(X), a.r = static_cast<const char *>(R), a.w = static_cast<const char *>(W);
    a.h = static_cast<char *>(H), a.y = static_cast<char *>(Y), a.scales = scales;
    a.M = M, a.N = (int)N;
    a.sx = x_stride, a.sr = r_stride, a.sh = h_stride, a.sy = y_stride;
    a.group_shift = 0;
    while (group && (1 << a.group_shift) < group) ++a.group_shift;
    a.n_groups = group ? (int)((N + group - 1) / group) : 1;
    a.eps = eps, a.inv_n = 1.0f / (float)N;
    // warps per row: `want` spans of 256 columns a warp
    const int64_t total = (N + 255) / 256;
    const int want = M < 296 ? 1 : 2;
    int64_t warps = (total + want - 1) / want;
    if (warps > kMaxRegThreads / 32) warps = kMaxRegThreads / 32;
    int64_t spans = (total + warps - 1) / warps;
    spans = spans <= 4 ? spans : spans <= 8 ? 8 : 0;
    if (spans > 0 && spans < 8) warps = (total + spans - 1) / spans;
    a.tpr = (int)warps * 32;
    int rpb = 1;
    if (M >= 296)
        while (rpb * 2 * a.tpr <= 64) rpb *= 2;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == DECA_F16 ? launch_out<DECA_F16>(a, out, v, (int)spans, rpb, st)
                             : launch_out<DECA_BF16>(a, out, v, (int)spans, rpb, st);
}
