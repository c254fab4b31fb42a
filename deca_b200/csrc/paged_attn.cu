// Entry points of the paged attention: argument rules, choice of the schedule, workspace.
#include <cmath>

#include "overlap.cuh"
#include "paged_attn.cuh"

namespace deca {
int paged_rows_ctas(int D, int mt, int sms);
size_t paged_rows_workspace(int D, int mt, int sms);
int paged_rows_launch(const deca_paged_attn_args &a, PagedArgs &g, int mt, bool cut, int sms, cudaStream_t st);
size_t paged_tiles_workspace(int D, int sms);
int paged_tiles_launch(const deca_paged_attn_args &a, PagedArgs &g, int sms, cudaStream_t st);

namespace {

bool tokens_ok(const deca_tokens &t) {
    return aligned_to(t.data, 16) && t.token_stride % 8 == 0 && t.head_stride % 8 == 0;
}
bool cache_ok(const deca_cache &c) {
    return aligned_to(c.data, 16) && c.page_stride % 8 == 0 && c.row_stride % 8 == 0 && c.head_stride % 8 == 0;
}

// 16 rows each of the streaming schedule
int row_tiles(const deca_paged_attn_args &a) { return (int64_t)a.max_q * (a.H_q / a.H_kv) <= 16 ? 1 : 2; }

// The tensor-core tiles take what has more than 32 query rows per request and key head, and from 17 rows on what the
// streaming schedule divides badly.  Measured with 17 .. 32 rows (D = 128, 8 key heads, streamed / tiles): few pairs of
// long contexts, 8 x 4000 keys 68 / 49 us, 1 x 8192 53 / 23, 9 x 1500 46 / 36 (D = 64: 1 x 8192 34 / 19, 4 x 4000 25 /
// 26), but 2 x 500 15.8 / 16.0; more pairs than CTAs, 64 x 2000 .. 8000 397 / 351, 100 x 0 .. 3000 202 / 170, but
// 200 x 0 .. 2000 233 / 239 and D = 64 64 x 2000 .. 8000 189 / 253.  Between them, 32 x 3000 88 / 120.
bool use_tiles(const deca_paged_attn_args &a, int sms) {
    const int64_t rows = (int64_t)a.max_q * (a.H_q / a.H_kv), pairs = (int64_t)a.B * a.H_kv;
    if (rows <= 16 || !(a.scale > 0.f)) return false;  // the tiles keep maxima of unscaled scores
    return rows > 32 || (2 * pairs <= sms && a.max_kv > 768) || (a.D == 128 && pairs > 2 * (int64_t)sms && a.max_kv > 2048);
}
// Whether the streaming schedule cuts items.  Whole, a (request, key head) pair is one CTA's and costs nothing but
// its keys; cut, the CTAs share the keys evenly, which costs 3 - 10 us of partial results and joining.  Measured
// (D = 128, 8 key heads, 16 rows, whole / cut): 16 x 2000 keys 28.3 / 31.8 us, 37 x 3000 72.9 / 75.2, 256 x 100 .. 500
// 66.8 / 72.8; but 4 x 4000 49 / 21, 1 x 8192 93 / 18, 64 x 0 .. 3000 90.6 / 77.8, 100 x 0 .. 1500 65.1 / 62.6, 100 x
// 1000 .. 4000 193 / 172; D = 64: 64 x 0 .. 4000 67.8 / 59.4.  More pairs than CTAs gain at any length where the last
// round is nearly empty (150 x 0 .. 3000, 2 key heads, 71.6 / 53.2), and with small CTAs (D = 64) or 32 rows only there:
// 100 x 0 .. 2000 (16 heads of 64) 76.8 / 85.5, 200 x 0 .. 2000 (32 rows) 225 / 294.
bool use_cuts(const deca_paged_attn_args &a, int sms) {
    if (a.max_kv <= 768) return false;
    const double pairs = (double)a.B * a.H_kv, ctas = paged_rows_ctas(a.D, row_tiles(a), sms);
    if (8 * pairs < 3 * ctas) return true;
    // microseconds of reading half of the longest contexts
    const double us = pairs * a.max_kv * a.D * 2.0 / 6.5e6;
    if (us > 36 && (pairs <= ctas || (a.D == 128 && row_tiles(a) == 1))) return true;
    return pairs > ctas && us * (std::ceil(pairs / ctas) * ctas / pairs - 1.0) > 15;  // the last round's idle share of them
}
// Tensor maps want strides that advance.  A dimension of one element may have any; a head stride of zero (one key head
// expanded to several) becomes a dimension of one element.
bool normalise(int64_t &stride, int64_t extent, int64_t any) {
    if (extent <= 1) stride = any;
    return stride > 0;
}
bool cache_strides(const deca_paged_attn_args &a, const deca_cache &c, long long &sp, long long &sr, long long &sh, int &heads) {
    int64_t p = c.page_stride, r = c.row_stride, h = c.head_stride;
    heads = a.H_kv > 1 && h == 0 ? 0 : 1;
    const bool ok = normalise(p, a.num_pages, a.D) && normalise(r, a.page_size, a.D) && normalise(h, heads ? a.H_kv : 1, a.D);
    sp = p, sr = r, sh = h;
    return ok;
}
bool query_strides(const deca_paged_attn_args &a, long long &st, long long &sh) {
    int64_t t = a.Q.token_stride, h = a.Q.head_stride;
    const bool ok = normalise(t, a.T, a.D) && normalise(h, a.H_q, a.D);
    st = t, sh = h;
    return ok;
}

// O may replace Q (an item's rows are read before the same rows are written) and must be apart from all else; the
// workspace from everything.
bool outputs_apart(const deca_paged_attn_args &a) {
    auto tokens = [&](const deca_tokens &t) { return region(t.data, 2 * a.D, a.T, 2 * t.token_stride, a.H_q, 2 * t.head_stride); };
    auto cache = [&](const deca_cache &c) {
        return region(c.data, 2 * a.D, a.num_pages, 2 * c.page_stride, a.page_size, 2 * c.row_stride, a.H_kv, 2 * c.head_stride);
    };
    const Region q = tokens(a.Q), o = tokens(a.O), ws = region(a.workspace, (int64_t)a.workspace_bytes);
    if (!regions_equal(q, o) && !regions_apart(q, o)) return false;
    for (const Region &r : {cache(a.K), cache(a.V), region(a.block_table, 4ll * a.table_width, a.B, 4 * a.table_stride), region(a.cu_q, 4 * (a.B + 1ll)),
                            region(a.kv_lens, 4ll * a.B)})
        if (!regions_apart(r, o) || !regions_apart(r, ws)) return false;
    return regions_apart(q, ws) && regions_apart(o, ws);
}

}  // namespace
}  // namespace deca

using namespace deca;

extern "C" int deca_paged_attn_check(const deca_paged_attn_args *a) {
    if (!a) return DECA_ERR_NULL;
    if (a->dtype != DECA_F16 && a->dtype != DECA_BF16) return DECA_ERR_UNSUPPORTED;
    if (a->D != 64 && a->D != 128) return DECA_ERR_UNSUPPORTED;
    if (a->B < 1 || a->H_q < 1 || a->H_kv < 1 || a->H_q % a->H_kv != 0 || a->H_q / a->H_kv > 128) return DECA_ERR_SHAPE;
    if (a->T < 0 || a->T > 2147483647ll || a->num_pages < 1 || a->num_pages > 2147483647ll) return DECA_ERR_SHAPE;
    if (a->page_size != 16 && a->page_size != 32 && a->page_size != 64 && a->page_size != 128 && a->page_size != 256)
        return DECA_ERR_SHAPE;
    if (a->table_width < 1 || a->table_stride < a->table_width) return DECA_ERR_SHAPE;
    if ((int64_t)a->table_width * a->page_size > 2147483647ll - 65536) return DECA_ERR_SHAPE;
    if (a->max_q < 0 || a->max_kv < 0) return DECA_ERR_SHAPE;
    if (!(a->scale == a->scale) || a->scale - a->scale != 0.f) return DECA_ERR_CONFIG;  // NaN or infinite
    if (!a->Q.data || !a->O.data || !a->K.data || !a->V.data || !a->block_table || !a->cu_q || !a->kv_lens) return DECA_ERR_NULL;
    if (!tokens_ok(a->Q) || !tokens_ok(a->O) || !cache_ok(a->K) || !cache_ok(a->V)) return DECA_ERR_ALIGN;
    long long sp, sr, sh;
    int heads;
    if (!cache_strides(*a, a->K, sp, sr, sh, heads) || !cache_strides(*a, a->V, sp, sr, sh, heads)) return DECA_ERR_ALIGN;
    if (!aligned_to(a->block_table, 4) || !aligned_to(a->cu_q, 4) || !aligned_to(a->kv_lens, 4)) return DECA_ERR_ALIGN;
    return DECA_OK;
}

extern "C" int deca_paged_attn_workspace_bytes(const deca_paged_attn_args *a, size_t *bytes) {
    if (!a || !bytes) return DECA_ERR_NULL;
    if ((a->D != 64 && a->D != 128) || a->H_kv < 1) return DECA_ERR_UNSUPPORTED;
    DeviceInfo di;
    if (int rc = current_device_info(&di)) return rc;
    *bytes = use_cuts(*a, di.sms) ? paged_rows_workspace(a->D, row_tiles(*a), di.sms) : 0;
    if (use_tiles(*a, di.sms) && paged_tiles_workspace(a->D, di.sms) > *bytes) *bytes = paged_tiles_workspace(a->D, di.sms);
    return DECA_OK;
}

extern "C" int deca_paged_attn(const deca_paged_attn_args *a, void *stream) {
    if (int rc = deca_paged_attn_check(a)) return rc;
    if (a->T == 0) return DECA_OK;
    if (!outputs_apart(*a)) return DECA_ERR_UNSUPPORTED;
    size_t need = 0;
    if (int rc = deca_paged_attn_workspace_bytes(a, &need)) return rc;
    if (need > 0 && !a->workspace) return DECA_ERR_NULL;
    if (!aligned_to(a->workspace, 256)) return DECA_ERR_ALIGN;
    if (a->workspace_bytes < need) return DECA_ERR_SCRATCH_LIMIT;
    DeviceInfo di;
    if (int rc = current_device_info(&di)) return rc;
    PagedArgs g = {};
    g.q = static_cast<const char *>(a->Q.data), g.q_st = a->Q.token_stride, g.q_sh = a->Q.head_stride;
    g.o = static_cast<char *>(a->O.data), g.o_st = a->O.token_stride, g.o_sh = a->O.head_stride;
    g.k = static_cast<const char *>(a->K.data), g.v = static_cast<const char *>(a->V.data);
    cache_strides(*a, a->K, g.k_sp, g.k_sr, g.k_sh, g.k_heads);
    cache_strides(*a, a->V, g.v_sp, g.v_sr, g.v_sh, g.v_heads);
    g.table = a->block_table, g.table_stride = a->table_stride, g.W = a->table_width;
    g.cu = a->cu_q, g.kv_lens = a->kv_lens;
    g.T = a->T, g.num_pages = a->num_pages, g.B = a->B, g.Hkv = a->H_kv, g.group = a->H_q / a->H_kv;
    while ((1 << g.page_shift) < a->page_size) ++g.page_shift;
    g.causal = a->causal ? 1 : 0;
    g.sl2 = a->scale * kLog2e;
    g.status = device_status_ptr();
    if (!g.status) return (int)cudaErrorUnknown;
    if (use_tiles(*a, di.sms) && query_strides(*a, g.q_st, g.q_sh)) {
        g.min_steps = 2;
        g.max_parts = 1 << 20;
        return paged_tiles_launch(*a, g, di.sms, static_cast<cudaStream_t>(stream));
    }
    return paged_rows_launch(*a, g, row_tiles(*a), use_cuts(*a, di.sms), di.sms, static_cast<cudaStream_t>(stream));
}
