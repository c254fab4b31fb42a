// Rotary positions (deca_rotary) and their fusion with the append to a paged cache
// (deca_rotary_append): q rotated into a tensor of its own, k rotated and v copied into the cache
// rows that the slots name, in one launch.
//
// The angle of pair i at position p is p * turns[i] modulo a turn, with turns[i] a 64-bit fixed-point
// fraction: the integer product wraps exactly where the angle does, so a position of a million loses
// nothing (an fp32 product would be off by 0.06 rad there) and no table of angles is read.  cos and sin
// are computed once per token into shared memory and shared by all heads: for 48 heads of 128 that is
// one sincospi per 96 elements.  What is left is a copy: every element is read once and written once.
#include "common.cuh"

namespace deca {
namespace {

constexpr int kMaxPairs = 128;
constexpr int kThreads = 256;

struct Turns {
    unsigned long long t[kMaxPairs];
};

struct RotArgs {
    const char *q, *k, *v;
    char *qo, *kc, *vc;
    long long q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh;  // elements
    long long kc_sp, kc_sr, kc_sh, vc_sp, vc_sr, vc_sh;
    const int *positions;
    const long long *slots;
    long long n_slots;  // num_pages * page_size
    int page_shift;     // log2(page_size)
    int Hq, Hkv;        // Hkv = 0: no append
    int D, rot;
    float amplitude;    // negative sign of the sine folded into `sine`
    float sine;
};

// V elements, 16 bytes (V = 8) or one element (V = 1)
template <int DT, int V>
__device__ __forceinline__ void load_part(float (&f)[V], const char *p) {
    if constexpr (V == 8) {
        uint32_t d[4];
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                     : "l"(p));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 x = Pack16<DT>::unpack(d[i]);
            f[2 * i] = x.x, f[2 * i + 1] = x.y;
        }
    } else if constexpr (DT == DECA_F16) {
        f[0] = __half2float(*reinterpret_cast<const __half *>(p));
    } else {
        f[0] = __bfloat162float(*reinterpret_cast<const __nv_bfloat16 *>(p));
    }
}
template <int DT, int V>
__device__ __forceinline__ void store_part(char *p, const float (&f)[V]) {
    if constexpr (V == 8) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(Pack16<DT>::pack(f[0], f[1]), Pack16<DT>::pack(f[2], f[3]),
                                                   Pack16<DT>::pack(f[4], f[5]), Pack16<DT>::pack(f[6], f[7]));
    } else if constexpr (DT == DECA_F16) {
        *reinterpret_cast<__half *>(p) = __float2half_rn(f[0]);
    } else {
        *reinterpret_cast<__nv_bfloat16 *>(p) = __float2bfloat16_rn(f[0]);
    }
}

// One unit of a head is two parts of V elements: unit u < rot / 2V holds V whole pairs, the others lie
// behind the rotated elements.
template <int DT, int V, int LAYOUT>
struct Unit {
    float a[V], b[V];
    static __device__ __forceinline__ int off_a(int u, int rot) {
        return (LAYOUT == DECA_ROT_HALF && u * 2 * V < rot) ? u * V : u * 2 * V;
    }
    static __device__ __forceinline__ int off_b(int u, int rot) {
        return (LAYOUT == DECA_ROT_HALF && u * 2 * V < rot) ? u * V + rot / 2 : u * 2 * V + V;
    }
    __device__ __forceinline__ void load(const char *head, int u, int rot) {
        load_part<DT, V>(a, head + 2 * off_a(u, rot));
        load_part<DT, V>(b, head + 2 * off_b(u, rot));
    }
    __device__ __forceinline__ void store(char *head, int u, int rot) const {
        store_part<DT, V>(head + 2 * off_a(u, rot), a);
        store_part<DT, V>(head + 2 * off_b(u, rot), b);
    }
    __device__ __forceinline__ void turn(const float2 *cs, int u) {
        if constexpr (LAYOUT == DECA_ROT_HALF || V == 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float2 w = cs[u * V + i];
                const float x = a[i], y = b[i];
                a[i] = x * w.x - y * w.y;
                b[i] = x * w.y + y * w.x;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 2) {  // pairs lie side by side within a part
                float2 w = cs[u * V + i / 2];
                float x = a[i], y = a[i + 1];
                a[i] = x * w.x - y * w.y;
                a[i + 1] = x * w.y + y * w.x;
                w = cs[u * V + V / 2 + i / 2];
                x = b[i], y = b[i + 1];
                b[i] = x * w.x - y * w.y;
                b[i + 1] = x * w.y + y * w.x;
            }
        }
    }
};

template <int DT, int V, int LAYOUT>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotArgs g, const __grid_constant__ Turns turns) {
    __shared__ float2 cs[kMaxPairs];
    using U = Unit<DT, V, LAYOUT>;
    const long long tok = blockIdx.x;
    const int per_head = g.D / (2 * V);
    const int n_units = (g.Hq + 2 * g.Hkv) * per_head;
    const int step = kThreads * gridDim.y;
    int i = blockIdx.y * kThreads + threadIdx.x;

    const char *src = nullptr;
    char *dst = nullptr;
    int u = 0;
    bool rotate = false;
    long long row_k = -1, row_v = -1;  // element offsets of the token's cache rows, -1: none
    if (g.Hkv > 0) {
        const long long slot = g.slots[tok];
        if (slot >= 0 && slot < g.n_slots) {
            const long long page = slot >> g.page_shift, row = slot & ((1ll << g.page_shift) - 1);
            row_k = page * g.kc_sp + row * g.kc_sr;
            row_v = page * g.vc_sp + row * g.vc_sr;
        }
    }
    auto place = [&](int idx) {  // unit idx of the token: heads of q, then k, then v
        int head = idx / per_head;
        u = idx - head * per_head;
        rotate = u * 2 * V < g.rot;
        if (head < g.Hq) {
            src = g.q + 2 * (tok * g.q_st + head * g.q_sh);
            dst = g.qo + 2 * (tok * g.qo_st + head * g.qo_sh);
            return;
        }
        head -= g.Hq;
        if (head < g.Hkv) {
            src = g.k + 2 * (tok * g.k_st + head * g.k_sh);
            dst = row_k >= 0 ? g.kc + 2 * (row_k + head * g.kc_sh) : nullptr;
        } else {
            head -= g.Hkv;
            src = g.v + 2 * (tok * g.v_st + head * g.v_sh);
            dst = row_v >= 0 ? g.vc + 2 * (row_v + head * g.vc_sh) : nullptr;
            rotate = false;
        }
    };
    // the first unit's loads are in flight while the angles are computed.  A v unit is copied, so its
    // parts need not follow the pairing of the rotation
    U x;
    if (i < n_units) {
        place(i);
        x.load(src, u, g.rot);
    }
    const long long pos = g.positions[tok];
    for (int p = threadIdx.x; p < g.rot / 2; p += kThreads) {
        const long long angle = (long long)((unsigned long long)pos * turns.t[p]);  // 2^63 = half a turn
        float s, c;
        sincospif((float)angle * 1.0842021724855044e-19f, &s, &c);
        cs[p] = make_float2(c * g.amplitude, s * g.sine);
    }
    __syncthreads();
    while (i < n_units) {
        if (rotate) x.turn(cs, u);
        if (dst) x.store(dst, u, g.rot);
        i += step;
        if (i < n_units) {
            place(i);
            x.load(src, u, g.rot);
        }
    }
}

int rotation_rules(int dtype, const deca_rotation *r) {
    if (!r || !r->turns) return DECA_ERR_NULL;
    if (dtype != DECA_F16 && dtype != DECA_BF16) return DECA_ERR_UNSUPPORTED;
    if (r->layout != DECA_ROT_HALF && r->layout != DECA_ROT_INTERLEAVED) return DECA_ERR_UNSUPPORTED;
    if (r->D < 2 || r->D > 2 * kMaxPairs || r->D % 2 != 0) return DECA_ERR_SHAPE;
    if (r->rot_dim < 2 || r->rot_dim > r->D || r->rot_dim % 2 != 0) return DECA_ERR_SHAPE;
    return DECA_OK;
}

bool vector_ok(const deca_tokens *t) {
    return aligned_to(t->data, 16) && t->token_stride % 8 == 0 && t->head_stride % 8 == 0;
}
bool vector_ok(const deca_cache *c) {
    return aligned_to(c->data, 16) && c->page_stride % 8 == 0 && c->row_stride % 8 == 0 && c->head_stride % 8 == 0;
}

template <int DT, int V>
void launch_layout(const RotArgs &g, const Turns &t, int layout, dim3 grid, cudaStream_t st) {
    if (layout == DECA_ROT_HALF)
        rotary_kernel<DT, V, DECA_ROT_HALF><<<grid, kThreads, 0, st>>>(g, t);
    else
        rotary_kernel<DT, V, DECA_ROT_INTERLEAVED><<<grid, kThreads, 0, st>>>(g, t);
}

int launch_rotary(int dtype, RotArgs &g, const deca_rotation *r, long long tokens, bool vec, cudaStream_t st) {
    if (tokens > 2147483647ll) return DECA_ERR_SHAPE;
    g.D = r->D, g.rot = r->rot_dim;
    g.amplitude = r->amplitude;
    g.sine = r->inverse ? -r->amplitude : r->amplitude;
    vec = vec && r->D % 16 == 0 && r->rot_dim % 16 == 0;
    Turns t;
    for (int i = 0; i < r->rot_dim / 2; ++i) t.t[i] = r->turns[i];
    for (int i = r->rot_dim / 2; i < kMaxPairs; ++i) t.t[i] = 0;
    // few tokens: the units of a token are shared by several CTAs
    const int units = (g.Hq + 2 * g.Hkv) * (r->D / (vec ? 16 : 2));
    int split = 1;
    while (tokens * split < 296 && split * kThreads < units && split < 64) split *= 2;
    const dim3 grid((unsigned)tokens, (unsigned)split);
    if (dtype == DECA_F16)
        vec ? launch_layout<DECA_F16, 8>(g, t, r->layout, grid, st) : launch_layout<DECA_F16, 1>(g, t, r->layout, grid, st);
    else
        vec ? launch_layout<DECA_BF16, 8>(g, t, r->layout, grid, st) : launch_layout<DECA_BF16, 1>(g, t, r->layout, grid, st);
    return (int)cudaGetLastError();
}

}  // namespace
}  // namespace deca

using namespace deca;

extern "C" int deca_rotary(int dtype, const deca_tokens *X, const deca_tokens *Y, const int32_t *positions,
                           int64_t tokens, int heads, const deca_rotation *rot, void *stream) {
    if (int rc = rotation_rules(dtype, rot)) return rc;
    if (!X || !Y) return DECA_ERR_NULL;
    if (tokens < 0 || heads < 1 || heads > 65536) return DECA_ERR_SHAPE;
    if (tokens == 0) return DECA_OK;
    if (!X->data || !Y->data || !positions) return DECA_ERR_NULL;
    if (!aligned_to(X->data, 2) || !aligned_to(Y->data, 2) || !aligned_to(positions, 4)) return DECA_ERR_ALIGN;
    RotArgs g = {};
    g.q = static_cast<const char *>(X->data), g.q_st = X->token_stride, g.q_sh = X->head_stride;
    g.qo = static_cast<char *>(Y->data), g.qo_st = Y->token_stride, g.qo_sh = Y->head_stride;
    g.positions = positions;
    g.Hq = heads;
    return launch_rotary(dtype, g, rot, tokens, vector_ok(X) && vector_ok(Y), static_cast<cudaStream_t>(stream));
}

extern "C" int deca_rotary_append(int dtype, const deca_tokens *Q, const deca_tokens *K, const deca_tokens *V,
                                  const deca_tokens *Q_out, const deca_cache *K_cache, const deca_cache *V_cache,
                                  const int32_t *positions, const int64_t *slots, int64_t tokens, int H_q, int H_kv,
                                  int64_t num_pages, int page_size, const deca_rotation *rot, void *stream) {
    if (int rc = rotation_rules(dtype, rot)) return rc;
    if (!Q || !K || !V || !Q_out || !K_cache || !V_cache) return DECA_ERR_NULL;
    if (tokens < 0 || H_q < 1 || H_kv < 1 || H_q > 65536 || H_kv > 65536) return DECA_ERR_SHAPE;
    if (num_pages < 1 || num_pages > (1ll << 40) || page_size < 1 || (page_size & (page_size - 1)) != 0 || page_size > (1 << 20))
        return DECA_ERR_SHAPE;
    if (tokens == 0) return DECA_OK;
    if (!Q->data || !K->data || !V->data || !Q_out->data || !K_cache->data || !V_cache->data || !positions || !slots)
        return DECA_ERR_NULL;
    if (!aligned_to(positions, 4) || !aligned_to(slots, 8) || !aligned_to(Q->data, 2) || !aligned_to(K->data, 2) ||
        !aligned_to(V->data, 2) || !aligned_to(Q_out->data, 2) || !aligned_to(K_cache->data, 2) || !aligned_to(V_cache->data, 2))
        return DECA_ERR_ALIGN;
    RotArgs g = {};
    g.q = static_cast<const char *>(Q->data), g.q_st = Q->token_stride, g.q_sh = Q->head_stride;
    g.k = static_cast<const char *>(K->data), g.k_st = K->token_stride, g.k_sh = K->head_stride;
    g.v = static_cast<const char *>(V->data), g.v_st = V->token_stride, g.v_sh = V->head_stride;
    g.qo = static_cast<char *>(Q_out->data), g.qo_st = Q_out->token_stride, g.qo_sh = Q_out->head_stride;
    g.kc = static_cast<char *>(K_cache->data), g.kc_sp = K_cache->page_stride, g.kc_sr = K_cache->row_stride, g.kc_sh = K_cache->head_stride;
    g.vc = static_cast<char *>(V_cache->data), g.vc_sp = V_cache->page_stride, g.vc_sr = V_cache->row_stride, g.vc_sh = V_cache->head_stride;
    g.positions = positions;
    g.slots = reinterpret_cast<const long long *>(slots);
    g.n_slots = num_pages * page_size;
    while ((1 << g.page_shift) < page_size) ++g.page_shift;
    g.Hq = H_q, g.Hkv = H_kv;
    const bool vec = vector_ok(Q) && vector_ok(K) && vector_ok(V) && vector_ok(Q_out) && vector_ok(K_cache) && vector_ok(V_cache);
    return launch_rotary(dtype, g, rot, tokens, vec, static_cast<cudaStream_t>(stream));
}
