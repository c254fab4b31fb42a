// Residual addition + RMSNorm with a 16-bit or an e4m3 output (deca_add_rmsnorm).
//
//   h = x + res;  y = h * rsqrt(sum h^2 / N + eps) * w;  out dt(h) and dt(y), or e4m3(y / s) with
//   s = max |y| / 448 over the row or a group of columns.
//
// One pass: a row's h stays in fp32 registers between the sum of squares and the output (8 elements
// per chunk, C chunks per thread), so every element is read once and written once, which is the floor
// of an HBM-bound operator: 8 bytes per element, 7 with the 8-bit output.  The row is spread over
// threads in interleaved 16-byte chunks as in rowwise.cu; the columns of a scale group (a multiple of 32)
// are then the chunks of 4 .. 32 neighbouring lanes, whose maximum takes shuffles alone.
// Rows beyond the registers of a CTA are streamed twice (three times for one scale a row).
#include "common.cuh"

namespace deca {
namespace {

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
    int group, n_groups;
    float eps, inv_n;
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
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

// Eight consecutive elements from column `col` on as fp32; element-wise with zeros behind the row's end
// where rows are not made of aligned 16-byte chunks.
template <int DT, bool VEC>
__device__ __forceinline__ void load8(float (&f)[8], const char *row, int col, int N, bool stream) {
    if constexpr (VEC) {
        uint32_t d[4];
        if (stream)
            asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                         : "l"(row + (size_t)col * 2));
        else
            asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                         : "l"(row + (size_t)col * 2));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = Pack16<DT>::unpack(d[i]);
            f[2 * i] = v.x, f[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = col + i < N ? load1<DT>(row + (size_t)(col + i) * 2) : 0.f;
    }
}

template <int DT, bool VEC>
__device__ __forceinline__ void store8(char *row, int col, int N, const float (&f)[8]) {
    if constexpr (VEC) {
        asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(row + (size_t)col * 2),
                     "r"(Pack16<DT>::pack(f[0], f[1])), "r"(Pack16<DT>::pack(f[2], f[3])),
                     "r"(Pack16<DT>::pack(f[4], f[5])), "r"(Pack16<DT>::pack(f[6], f[7]))
                     : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < N) store1<DT>(row + (size_t)(col + i) * 2, f[i]);
    }
}

// Two values to e4m3 (round to nearest even, saturating, NaN kept), the first in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t v;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(v) : "f"(hi), "f"(lo));
    return v;
}

template <bool VEC>
__device__ __forceinline__ void store_e4m3(char *row, int col, int N, const float (&y)[8], float inv) {
    uint32_t lo = e4m3x2(y[0] * inv, y[1] * inv) | (e4m3x2(y[2] * inv, y[3] * inv) << 16);
    uint32_t hi = e4m3x2(y[4] * inv, y[5] * inv) | (e4m3x2(y[6] * inv, y[7] * inv) << 16);
    if constexpr (VEC) {
        asm volatile("st.global.cs.v2.u32 [%0], {%1,%2};" ::"l"(row + col), "r"(lo), "r"(hi) : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < N) row[col + i] = (char)(((i < 4 ? lo : hi) >> (8 * (i & 3))) & 0xFFu);
    }
}

__device__ __forceinline__ float abs_max8(const float (&y)[8]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(y[i]));
    return m;
}

// Scale and its inverse of a group whose largest |y| is `m`.
__device__ __forceinline__ void scale_of(float m, float &s, float &inv) {
    s = m * (1.0f / kE4m3Max);
    inv = s >= kMinScale ? 1.0f / s : 0.f;
}

// One chunk of a grouped e4m3 output: maximum over the lanes that share the group, scale, store.
// Called by all lanes of a warp; `col` is ordered by lane and group / 8 lanes share a group.
template <bool VEC>
__device__ __forceinline__ void store_grouped(const AddNormArgs &a, long long row, char *yrow, int col, bool live,
                                              const float (&y)[8]) {
    float m = live ? abs_max8(y) : 0.f;
    for (int s = a.group >> 4; s >= 1; s >>= 1) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, s));
    float scale, inv;
    scale_of(m, scale, inv);
    if (live) {
        if (col % a.group == 0) a.scales[row * a.n_groups + col / a.group] = scale;
        store_e4m3<VEC>(yrow, col, a.N, y, inv);
    }
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

// The row in registers: C chunks of eight elements per thread, `rpb` rows per CTA.
template <int DT, int OUT, int C, bool VEC>
__global__ void add_rmsnorm_reg_kernel(const AddNormArgs a) {
    __shared__ float red[2][32];
    const int t = threadIdx.x % a.tpr, rb = threadIdx.x / a.tpr;
    const int lane = threadIdx.x & 31, wr = t >> 5, nw = a.tpr >> 5;
    long long row = (long long)blockIdx.x * (blockDim.x / a.tpr) + rb;
    const bool live_row = row < a.M;  // the threads of a row behind the last one take part in the barriers only
    if (!live_row) row = 0;
    const char *xrow = a.x + row * a.sx * 2, *rrow = a.r + row * a.sr * 2;
    char *hrow = a.h + row * a.sh * 2, *yrow = a.y + row * a.sy * (OUT == DECA_OUT_SAME ? 2 : 1);

    float h[C][8];
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int col = (c * a.tpr + t) * 8;
        float r[8];
        if (live_row && col < a.N) {
            load8<DT, VEC>(h[c], xrow, col, a.N, true);
            load8<DT, VEC>(r, rrow, col, a.N, true);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = r[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) h[c][i] += r[i];
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(h[c][i], h[c][i], ss);
    ss = row_reduce<false>(ss, red[0], nw, rb * nw, wr, lane);
    const float rs = rsqrtf(fmaf(ss, a.inv_n, a.eps));

    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int col = (c * a.tpr + t) * 8;
        const bool live = live_row && col < a.N;
        if (live) store8<DT, VEC>(hrow, col, a.N, h[c]);
        float w[8];
        if (live) {
            load8<DT, VEC>(w, a.w, col, a.N, false);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = h[c][i] * rs * w[i];
        }
        if constexpr (OUT == DECA_OUT_SAME) {
            if (live) store8<DT, VEC>(yrow, col, a.N, h[c]);
        } else if (a.group > 0) {
            store_grouped<VEC>(a, row, yrow, col, live, h[c]);
        } else if (live) {
            amax = max_nan(amax, abs_max8(h[c]));
        }
    }
    if constexpr (OUT == DECA_OUT_E4M3) {
        if (a.group == 0) {
            amax = row_reduce<true>(amax, red[1], nw, rb * nw, wr, lane);
            float scale, inv;
            scale_of(amax, scale, inv);
            if (live_row && t == 0) a.scales[row] = scale;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int col = (c * a.tpr + t) * 8;
                if (live_row && col < a.N) store_e4m3<VEC>(yrow, col, a.N, h[c], inv);
            }
        }
    }
}

// Rows of any length: the row is read once for the sum of squares, (one scale a row) once for the
// maximum and once for the output; re-reads come from L2.
template <int DT, int OUT, bool VEC>
__global__ void add_rmsnorm_stream_kernel(const AddNormArgs a) {
    __shared__ float red[2][32];
    const int t = threadIdx.x, lane = t & 31, wr = t >> 5, nw = blockDim.x >> 5;
    const long long row = blockIdx.x;
    const char *xrow = a.x + row * a.sx * 2, *rrow = a.r + row * a.sr * 2;
    char *hrow = a.h + row * a.sh * 2, *yrow = a.y + row * a.sy * (OUT == DECA_OUT_SAME ? 2 : 1);
    const int span = (int)blockDim.x * 8;
    auto load_h = [&](float (&h)[8], int col) {
        float r[8];
        load8<DT, VEC>(h, xrow, col, a.N, false);
        load8<DT, VEC>(r, rrow, col, a.N, false);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] += r[i];
    };
    auto load_y = [&](float (&y)[8], int col, float rs) {
        float w[8];
        load8<DT, VEC>(w, a.w, col, a.N, false);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * rs * w[i];
    };
    float ss = 0.f;
    for (int base = 0; base < a.N; base += span) {
        const int col = base + t * 8;
        if (col < a.N) {
            float h[8];
            load_h(h, col);
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(h[i], h[i], ss);
        }
    }
    ss = row_reduce<false>(ss, red[0], nw, 0, wr, lane);
    const float rs = rsqrtf(fmaf(ss, a.inv_n, a.eps));
    float scale = 0.f, inv = 0.f;
    if constexpr (OUT == DECA_OUT_E4M3) {
        if (a.group == 0) {
            float amax = 0.f;
            for (int base = 0; base < a.N; base += span) {
                const int col = base + t * 8;
                if (col < a.N) {
                    float y[8];
                    load_h(y, col);
                    load_y(y, col, rs);
                    amax = max_nan(amax, abs_max8(y));
                }
            }
            amax = row_reduce<true>(amax, red[1], nw, 0, wr, lane);
            scale_of(amax, scale, inv);
            if (t == 0) a.scales[row] = scale;
        }
    }
    // every element is read again and then written by the same thread, so H may be X or R
    for (int base = 0; base < a.N; base += span) {
        const int col = base + t * 8;
        const bool live = col < a.N;
        float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (live) {
            load_h(y, col);
            store8<DT, VEC>(hrow, col, a.N, y);
            load_y(y, col, rs);
        }
        if constexpr (OUT == DECA_OUT_SAME) {
            if (live) store8<DT, VEC>(yrow, col, a.N, y);
        } else if (a.group > 0) {
            store_grouped<VEC>(a, row, yrow, col, live, y);
        } else if (live) {
            store_e4m3<VEC>(yrow, col, a.N, y, inv);
        }
    }
}

constexpr int kMaxChunks = 8;
constexpr int kMaxRegThreads = 512;

template <int DT, int OUT, bool VEC>
int launch(const AddNormArgs &a0, int chunks, int rpb, cudaStream_t st) {
    AddNormArgs a = a0;
    if (chunks == 0) {
        if (a.M > 2147483647ll) return DECA_ERR_SHAPE;
        add_rmsnorm_stream_kernel<DT, OUT, VEC><<<(unsigned)a.M, 512, 0, st>>>(a);
        return (int)cudaGetLastError();
    }
    const long long grid = (a.M + rpb - 1) / rpb;
    if (grid > 2147483647ll) return DECA_ERR_SHAPE;
    const unsigned g = (unsigned)grid, threads = (unsigned)(a.tpr * rpb);
    switch (chunks) {
        case 1: add_rmsnorm_reg_kernel<DT, OUT, 1, VEC><<<g, threads, 0, st>>>(a); break;
        case 2: add_rmsnorm_reg_kernel<DT, OUT, 2, VEC><<<g, threads, 0, st>>>(a); break;
        case 4: add_rmsnorm_reg_kernel<DT, OUT, 4, VEC><<<g, threads, 0, st>>>(a); break;
        default: add_rmsnorm_reg_kernel<DT, OUT, 8, VEC><<<g, threads, 0, st>>>(a); break;
    }
    return (int)cudaGetLastError();
}

template <int DT>
int launch_out(const AddNormArgs &a, int out, bool vec, int chunks, int rpb, cudaStream_t st) {
    if (out == DECA_OUT_SAME)
        return vec ? launch<DT, DECA_OUT_SAME, true>(a, chunks, rpb, st) : launch<DT, DECA_OUT_SAME, false>(a, chunks, rpb, st);
    return vec ? launch<DT, DECA_OUT_E4M3, true>(a, chunks, rpb, st) : launch<DT, DECA_OUT_E4M3, false>(a, chunks, rpb, st);
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
    const bool rows_vec = M == 1 || (x_stride % 8 == 0 && r_stride % 8 == 0 && h_stride % 8 == 0 && y_stride % 8 == 0);
    const bool vec = N % 8 == 0 && rows_vec && aligned_to(X, 16) && aligned_to(R, 16) && aligned_to(W, 16) &&
                     aligned_to(H, 16) && aligned_to(Y, 8 * out_bytes);
    AddNormArgs a;
    a.x = static_cast<const char *>(X), a.r = static_cast<const char *>(R), a.w = static_cast<const char *>(W);
    a.h = static_cast<char *>(H), a.y = static_cast<char *>(Y), a.scales = scales;
    a.M = M, a.N = (int)N;
    a.sx = x_stride, a.sr = r_stride, a.sh = h_stride, a.sy = y_stride;
    a.group = group;
    a.n_groups = group ? (int)((N + group - 1) / group) : 1;
    a.eps = eps, a.inv_n = 1.0f / (float)N;
    // threads per row: four chunks a thread where there are rows to fill the SMs, one where there are few
    int tpr = 32;
    const int want = M < 296 ? 1 : 4;
    while (tpr < kMaxRegThreads && (int64_t)tpr * 8 * want < N) tpr *= 2;
    int64_t chunks = (N + (int64_t)tpr * 8 - 1) / ((int64_t)tpr * 8);
    chunks = chunks <= 1 ? 1 : chunks <= 2 ? 2 : chunks <= 4 ? 4 : chunks <= kMaxChunks ? 8 : 0;
    a.tpr = tpr;
    int rpb = 1;
    if (M >= 296)
        while (rpb * tpr < 64) rpb *= 2;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == DECA_F16 ? launch_out<DECA_F16>(a, out, vec, (int)chunks, rpb, st)
                             : launch_out<DECA_BF16>(a, out, vec, (int)chunks, rpb, st);
}
