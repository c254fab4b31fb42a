// Rotary positions (deca_rotary) and their fusion with the append to a paged cache
// (deca_rotary_append): q rotated into a tensor of its own, k rotated and v copied into the cache
// rows that the slots name, in one launch.
//
// The angle of pair i at position p is p * turns[i] modulo a turn, with turns[i] a 64-bit fixed-point
// fraction: the integer product wraps exactly where the angle does, so a position of a million loses
// nothing (an fp32 product would be off by 0.06 rad there) and no table of angles is read.  cos and sin
// are computed once per token into shared memory and shared by all heads: for 48 heads of 128 that is
// one sincospi per 96 elements.  What is left is a copy: every element is read once and written once.
//
// Bound by HBM: 8192 tokens of 32 + 2 x 8 heads of 128 in fp16 (201 MB) 36.3 us = 5.54 TB/s, 84 % of the measured copy
// rate; 4099 tokens of 24 heads 10.6 us; 8 tokens 2.7 us (launch latency; a token's heads are then shared by several
// CTAs).  A CTA per token without the walk took 40 us, with one unit in flight per thread instead of three 53.
#include "common.cuh"
#include "overlap.cuh"
#include "ptx.cuh"

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
    long long tokens;
    int D, rot;
    float amplitude;    // negative sign of the sine folded into `sine`
    float sine;
};

// V elements as they lie in memory: 16 bytes (V = 8) or one element (V = 1)
template <int V>
struct Raw;
template <>
struct Raw<8> {
    uint32_t w[4];
    __device__ __forceinline__ void load(const char *p) {
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "l"(p));
    }
    __device__ __forceinline__ void store(char *p) const { *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]); }
    template <int DT>
    __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 x = Pack16<DT>::unpack(w[i]);
            f[2 * i] = x.x, f[2 * i + 1] = x.y;
        }
    }
    template <int DT>
    __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = Pack16<DT>::pack(f[2 * i], f[2 * i + 1]);
    }
};
template <>
struct Raw<1> {
    uint16_t w;
    __device__ __forceinline__ void load(const char *p) { w = *reinterpret_cast<const uint16_t *>(p); }
    __device__ __forceinline__ void store(char *p) const { *reinterpret_cast<uint16_t *>(p) = w; }
    template <int DT>
    __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = Pack16<DT>::unpack(w).x; }
    template <int DT>
    __device__ __forceinline__ void set(const float (&f)[1]) { w = (uint16_t)Pack16<DT>::pack(f[0], 0.f); }
};

// Turns the pairs of one unit; cs: the first of its V angles.
template <int DT, int V, int LAYOUT>
__device__ __forceinline__ void turn(Raw<V> &ra, Raw<V> &rb, const float2 *cs) {
    float a[V], b[V];
    ra.template get<DT>(a);
    rb.template get<DT>(b);
    if constexpr (LAYOUT == DECA_ROT_HALF || V == 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 w = cs[i];
            const float x = a[i], y = b[i];
            a[i] = x * w.x - y * w.y;
            b[i] = x * w.y + y * w.x;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) {  // pairs lie side by side within a part
            float2 w = cs[i / 2];
            float x = a[i], y = a[i + 1];
            a[i] = x * w.x - y * w.y;
            a[i + 1] = x * w.y + y * w.x;
            w = cs[V / 2 + i / 2];
            x = b[i], y = b[i + 1];
            b[i] = x * w.x - y * w.y;
            b[i + 1] = x * w.y + y * w.x;
        }
    }
    ra.template set<DT>(a);
    rb.template set<DT>(b);
}

constexpr int kUnits = 3;  // units of a thread whose loads are issued together

// A CTA takes every gridDim.x-th token (or a share of its heads, gridDim.y of them).  A unit is two parts of V
// elements of a head: V whole pairs, or 2 V elements behind the rotated ones; a thread keeps its place within
// the head and walks over the heads of q, then k, then v, so it needs one division.  A token's first units are on
// their way while its angles are computed.
template <int DT, int V, int LAYOUT>
__global__ void __launch_bounds__(kThreads, 5) rotary_kernel(const RotArgs g, const __grid_constant__ Turns turns) {
    __shared__ float2 angles[2][kMaxPairs];  // of two tokens in turn: one barrier per token
    const int per_head = g.D / (2 * V);
    const int at = blockIdx.y * blockDim.x + threadIdx.x;  // blockDim.x is a multiple of per_head
    const int u = at % per_head, step = (int)(blockDim.x * gridDim.y) / per_head;
    const bool rotated = u * 2 * V < g.rot;
    const bool split = LAYOUT == DECA_ROT_HALF && rotated;
    const int off_a = split ? u * V : u * 2 * V, off_b = split ? u * V + g.rot / 2 : u * 2 * V + V;
    const int heads = g.Hq + 2 * g.Hkv;
    const unsigned long long my_turn = (int)threadIdx.x < g.rot / 2 ? turns.t[threadIdx.x] : 0ull;
    float2 *cs = angles[0];

    for (long long tok = blockIdx.x; tok < g.tokens; tok += gridDim.x) {
        auto source = [&](int head) -> const char * {
            if (head < g.Hq) return g.q + 2 * (tok * g.q_st + head * g.q_sh);
            head -= g.Hq;
            if (head < g.Hkv) return g.k + 2 * (tok * g.k_st + head * g.k_sh);
            return g.v + 2 * (tok * g.v_st + (head - g.Hkv) * g.v_sh);
        };
        Raw<V> a[kUnits], b[kUnits];
        int head = at / per_head;
        auto load = [&]() {
#pragma unroll
            for (int i = 0; i < kUnits; ++i)
                if (head + i * step < heads) {
                    const char *src = source(head + i * step);
                    a[i].load(src + 2 * off_a);
                    b[i].load(src + 2 * off_b);
                }
        };
        const long long pos = g.positions[tok];
        const long long slot = g.Hkv > 0 ? g.slots[tok] : -1;
        load();
        for (int p = threadIdx.x; p < g.rot / 2; p += blockDim.x) {
            const unsigned long long turn = p < (int)blockDim.x ? my_turn : turns.t[p];
            const long long angle = (long long)((unsigned long long)pos * turn);  // 2^63 = half a turn
            float s, c;
            sincospif((float)angle * 1.0842021724855044e-19f, &s, &c);
            cs[p] = make_float2(c * g.amplitude, s * g.sine);
        }
        long long row_k = -1, row_v = -1;  // element offsets of the token's cache rows, -1: none
        if (slot >= 0 && slot < g.n_slots) {
            const long long page = slot >> g.page_shift, row = slot & ((1ll << g.page_shift) - 1);
            row_k = page * g.kc_sp + row * g.kc_sr;
            row_v = page * g.vc_sp + row * g.vc_sr;
        }
        __syncthreads();
        while (true) {
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                int h = head + i * step;
                if (h >= heads) break;
                char *dst;
                if (h < g.Hq) {
                    dst = g.qo + 2 * (tok * g.qo_st + h * g.qo_sh);
                } else if ((h -= g.Hq) < g.Hkv) {
                    dst = row_k >= 0 ? g.kc + 2 * (row_k + h * g.kc_sh) : nullptr;
                } else {
                    dst = row_v >= 0 ? g.vc + 2 * (row_v + (h - g.Hkv) * g.vc_sh) : nullptr;
                }
                if (rotated && head + i * step < g.Hq + g.Hkv) turn<DT, V, LAYOUT>(a[i], b[i], cs + u * V);
                if (dst) {
                    a[i].store(dst + 2 * off_a);
                    b[i].store(dst + 2 * off_b);
                }
            }
            head += kUnits * step;
            if (head >= heads) break;
            load();
        }
        cs = cs == angles[0] ? angles[1] : angles[0];
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

Region region_of(const deca_tokens *t, int64_t tokens, int heads, int D) {
    return region(t->data, 2 * (int64_t)D, tokens, 2 * t->token_stride, heads, 2 * t->head_stride);
}

template <int DT, int V>
void launch_layout(const RotArgs &g, const Turns &t, int layout, dim3 grid, unsigned threads, cudaStream_t st) {
    if (layout == DECA_ROT_HALF)
        rotary_kernel<DT, V, DECA_ROT_HALF><<<grid, threads, 0, st>>>(g, t);
    else
        rotary_kernel<DT, V, DECA_ROT_INTERLEAVED><<<grid, threads, 0, st>>>(g, t);
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
    const int per_head = r->D / (vec ? 16 : 2);
    const int heads = g.Hq + 2 * g.Hkv;
    // Threads: as few groups of a head's units as cover the heads in whole rounds, about `want` units each
    const int most = kThreads / per_head;  // heads that a CTA of full size takes at once
    const int want = tokens < 296 ? 1 : kUnits;
    int at_once = (heads + want - 1) / want;
    if (at_once * per_head < 64) at_once = (63 + per_head) / per_head;  // the angles want two warps
    if (at_once > most) at_once = most;
    // few tokens: the heads of a token are shared by several CTAs
    int split = 1;
    while (tokens * split < 296 && split * at_once < heads && split < 64) split *= 2;
    g.tokens = tokens;
    DeviceInfo di;
    if (int rc = current_device_info(&di)) return rc;
    const int resident = di.sms * (40 / ((at_once * per_head + 31) / 32));  // CTAs that run at once: 40 warps an SM
    const dim3 grid((unsigned)(tokens < resident ? tokens : resident), (unsigned)split);
    const unsigned threads = (unsigned)(at_once * per_head);
    if (dtype == DECA_F16)
        vec ? launch_layout<DECA_F16, 8>(g, t, r->layout, grid, threads, st) : launch_layout<DECA_F16, 1>(g, t, r->layout, grid, threads, st);
    else
        vec ? launch_layout<DECA_BF16, 8>(g, t, r->layout, grid, threads, st) : launch_layout<DECA_BF16, 1>(g, t, r->layout, grid, threads, st);
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
    // a pair is read and written by one thread, so Y may be X
    const Region x = region_of(X, tokens, heads, rot->D), y = region_of(Y, tokens, heads, rot->D);
    if ((!regions_equal(x, y) && !regions_apart(x, y)) || !regions_apart(y, region(positions, 4 * tokens))) return DECA_ERR_UNSUPPORTED;
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
    {
        const int D = rot->D;
        auto cache = [&](const deca_cache *c) {
            return region(c->data, 2 * (int64_t)D, num_pages, 2 * c->page_stride, page_size, 2 * c->row_stride, H_kv, 2 * c->head_stride);
        };
        const Region q = region_of(Q, tokens, H_q, D), k = region_of(K, tokens, H_kv, D), v = region_of(V, tokens, H_kv, D);
        const Region out = region_of(Q_out, tokens, H_q, D), kc = cache(K_cache), vc = cache(V_cache);
        const Region pos = region(positions, 4 * tokens), slot = region(slots, 8 * tokens);
        if (!regions_equal(q, out) && !regions_apart(q, out)) return DECA_ERR_UNSUPPORTED;
        if (!regions_apart(out, kc) || !regions_apart(out, vc) || !regions_apart(kc, vc)) return DECA_ERR_UNSUPPORTED;
        for (const Region &in : {k, v, pos, slot})
            if (!regions_apart(in, out)) return DECA_ERR_UNSUPPORTED;
        for (const Region &in : {q, k, v, pos, slot})
            if (!regions_apart(in, kc) || !regions_apart(in, vc)) return DECA_ERR_UNSUPPORTED;
    }
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
