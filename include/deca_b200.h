/*
 * deca_b200 -- C ABI of the B200 (sm_100a) kernels behind DeCA's operator hot path.
 *
 * The reference (BenkangPeng/Deca) has no C interface: each (shape, config) is generated
 * as TIR, compiled by TVM + nvcc and called as `load_module(path)["main"](*tensors)`
 * (src/RuntimeMod.py:104-109, :169-170, :204-205).  The entry points below are what a
 * binding for that call would bind instead: one per kernel family, the config passed as
 * a plain struct that mirrors the reference's config dataclass.
 *
 * Conventions
 *   - every function returns an int status: 0 ok; < 0 argument error found on the host
 *     (DECA_ERR_*), nothing was launched; > 0 a cudaError_t / CUresult value, or
 *     DECA_ERR_DEVICE_TIMEOUT when a kernel gave up on a bounded wait.
 *   - pointers are device pointers unless the name says host; the caller owns every
 *     buffer; the library allocates no device memory.
 *   - `stream` is a cudaStream_t passed as void* (0 = legacy default stream).
 *   - launches are asynchronous; nothing here synchronises the device.
 *   - thread safety: calls may come from several host threads.
 */
#ifndef DECA_B200_H
#define DECA_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DECA_OK 0
#define DECA_ERR_NULL (-1)        /* a required pointer is null */
#define DECA_ERR_SHAPE (-2)       /* non-positive or unsupported extent */
#define DECA_ERR_ALIGN (-3)       /* pointer or row pitch not aligned for the vector width / TMA */
#define DECA_ERR_CONFIG (-4)      /* config rejected by the check_config rules */
#define DECA_ERR_UNSUPPORTED (-5) /* op / dtype / mode not built; serving operators: an output over another buffer of the call */
#define DECA_ERR_SCRATCH_LIMIT (-6) /* the problem needs more scratch memory than the built-in buffer holds */
#define DECA_ERR_DEVICE_TIMEOUT 100001 /* a kernel's bounded wait ran out (see deca_last_device_status) */

enum { DECA_F16 = 0, DECA_BF16 = 1 };
enum { DECA_SOFTMAX = 0, DECA_RMSNORM = 1 };
enum { DECA_ROW_REG = 0, DECA_ROW_TWOPASS = 1, DECA_ROW_TMA = 2, DECA_ROW_CLUSTER = 3 };

/* Library version string, e.g. "deca_b200 0.1 (sm_100a)". */
const char *deca_version(void);

/* Text for a status returned by any function of this header. */
const char *deca_status_string(int status);

/* Kernels that wait on hardware barriers (bulk-copy pipelines, tensor-core pipelines) bound
 * every wait; a kernel that gives up records DECA_ERR_DEVICE_TIMEOUT, the site and the block
 * in a device status word and returns normally.  This call synchronises the device, copies
 * that word (0 = no timeout since the last clear) and optionally clears it.
 * The reference has no counterpart: its kernels have no device-side waits on barriers. */
int deca_last_device_status(int *code, int *where, int *block, int clear);

/* Diagnostics: copies the first n (<= 16) 32-bit words of the device status record: code, where,
 * block, reserved, then twelve per-role words (site << 16 | loop index) written by the roles of
 * block (0, 0) that left a bounded wait unsuccessfully.  Synchronises the device.
 * No counterpart in the reference. */
int deca_device_status_words(unsigned int *out, int n);

/* Self-test of the bounded-wait path: launches one small CTA (no bulk copies, no tensor cores)
 * in which a thread waits on a barrier that nothing arrives on, gives up after `limit_us`
 * microseconds (1 .. 100 000), raises the CTA's abort flag and records DECA_ERR_DEVICE_TIMEOUT
 * with site 0x7E57, as the pipelined kernels do when a wait of theirs runs out; a second thread
 * waiting with the kernels' 1 s limit has to leave through the abort flag.  The kernel then
 * returns normally and the context stays usable.  Read the outcome with deca_last_device_status
 * (clear = 1) or deca_device_status_words (words 4 and 5: how long the two threads waited, in
 * microseconds).  No counterpart in the reference. */
int deca_selftest_bounded_wait(unsigned int limit_us, void *stream);

/* ---------------------------------------------------------------------------------------
 * Row-wise softmax / RMSNorm over X[M, N] (row-major, 16-bit), reduction over N.
 * Replaces the kernels generated by make_rowwise (src/kernels/rowwise_tir.py:99-391).
 * The struct mirrors RowConfig (rowwise_tir.py:42-61).
 * ------------------------------------------------------------------------------------- */
typedef struct {
    int threads_per_row; /* multiple of 32; threads_per_row * rows_per_block <= 1024 */
    int rows_per_block;  /* rows sharing one CTA; must divide M (REG, TWOPASS).
                            TMA: independent row groups per persistent CTA (<= 15) */
    int vec;             /* elements per access: 8 (16 bytes), 4 (8 bytes) or 2 (4 bytes) */
    int mode;            /* DECA_ROW_REG: row cached in registers, read once;
                            DECA_ROW_TWOPASS: row streamed twice (online max/sum first);
                            DECA_ROW_TMA: persistent CTAs, rows streamed through shared-memory
                            rings with bulk copies (threads_per_row a power of two <= 512,
                            vec 8, (unroll + 2) * rows_per_block rows must fit shared memory);
                            DECA_ROW_CLUSTER: a thread-block cluster of `unroll` CTAs shares a row, every
                            CTA (threads_per_row threads, rows_per_block = 1) caches a contiguous slice
                            of it in registers (<= 8 chunks per thread) and the row statistics are
                            combined through distributed shared memory: long rows in one pass */
    int unroll;          /* TWOPASS: chunks in flight per iteration (1, 2 or 4);
                            TMA: input ring slots (rows in flight) per group, 1..8;
                            CLUSTER: CTAs per cluster (2, 4 or 8) */
    int hint;            /* non-zero: no-allocate / evict-first loads and streaming stores */
} deca_row_cfg;

/* Host-only mirror of check_config (rowwise_tir.py:88-96) plus this library's limits
 * (REG mode holds at most 32 chunks per thread, TMA mode at most 16).  Returns DECA_OK or DECA_ERR_*. */
int deca_rowwise_check_config(int op, int dtype, int64_t M, int64_t N, const deca_row_cfg *cfg);

/* Y = softmax(X, -1)                       (op = DECA_SOFTMAX, W ignored, may be null)
 * Y = dt(f32(dt(X * rsqrt(mean(X^2)+eps))) * W)   (op = DECA_RMSNORM, W[N])
 * fp32 math, 16-bit I/O.  X, Y (and W) must be aligned to vec * 2 bytes and N % vec == 0.
 * cfg == null selects a default config for the shape.
 * Replaces runtime_mod["main"](x[, w], y) of a row-wise kernel (RuntimeMod.py:204-208). */
int deca_rowwise(int op, int dtype, const void *X, const void *W, void *Y, int64_t M, int64_t N, float eps,
                 const deca_row_cfg *cfg, void *stream);

/* deca_rowwise that also writes, per row, the two fp32 statistics the kernel reduced the row to:
 * stats[2 * row], stats[2 * row + 1] = (row max * log2 e, 1 / sum of exponentials) for softmax,
 * (rsqrt(mean x^2 + eps), sum x^2) for RMSNorm.  They are the only quantities of these kernels
 * computed in fp32 across a row; everything after them is element-wise arithmetic and rounding to
 * the 16-bit type, so a checker can compare the statistics with an exact computation at fp32
 * accuracy, free of the 16-bit rounding of the outputs.  `stats` is a device buffer of 2 * M floats,
 * 8-byte aligned.  Every mode but DECA_ROW_TMA (DECA_ERR_UNSUPPORTED there).
 * Same kernels and same outputs as deca_rowwise.  No counterpart in the reference (a checking aid). */
int deca_rowwise_stats(int op, int dtype, const void *X, const void *W, void *Y, float *stats, int64_t M, int64_t N,
                       float eps, const deca_row_cfg *cfg, void *stream);

/* The config deca_rowwise uses when cfg == null. */
int deca_rowwise_default_config(int op, int dtype, int64_t M, int64_t N, deca_row_cfg *out);

/* ---------------------------------------------------------------------------------------
 * 16-bit tensor-core GEMM  C[M,N] = A[M,K] @ B[K,N], all row-major, fp16 or bf16 in and out,
 * fp32 accumulation (tcgen05.mma into tensor memory).
 * Replaces the kernel generated by make_gemm_tc (src/kernels/gemm_tir.py:123-386); the struct
 * takes the place of GemmConfig (gemm_tir.py:42-76) with the tile space of the tcgen05 kernel.
 * ------------------------------------------------------------------------------------- */
typedef struct {
    int BM;        /* tile rows per CTA: 128, or 256 (two MMAs per k step share the B tile) */
    int BN;        /* tile columns: 64, 128 or 256 */
    int BK;        /* K depth of one pipeline stage: 64 */
    int stages;    /* TMA -> MMA shared-memory ring depth, 2..8 */
    int raster;    /* tile rows per rasterisation group (>= 1) */
    int epi_smem;  /* non-zero: C leaves through shared memory and TMA stores; 0: direct stores */
    int cta_group; /* 1, or 2 = CTA pairs (tcgen05 cta_group::2) on a (2 BM) x BN tile: BM = 128 or 256 rows
                      per CTA, BN = 128 or 256, epi_smem = 1, no stream_k */
    int acc_bufs;  /* tensor-memory accumulators, 1 or 2 (acc_bufs * BM/128 * BN <= 512 columns) */
    int stream_k;  /* 1: when whole tiles would fill the last wave of CTAs to less than 95 %, the k
                      blocks of the last tiles are cut into equal shares, one per SM (needs scratch
                      memory: deca_gemm16_ws); 0: whole tiles only */
    int acc_f16;   /* 1: accumulate in fp16 instead of fp32 (the accumulator type of tcgen05.mma.kind::f16
                      set to f16), the counterpart of GemmConfig.acc_f16 (gemm_tir.py:52-58): fp16 inputs,
                      cta_group = 1, no stream_k.  An fp16 accumulator still takes one 32-bit tensor-memory
                      column per value, so it frees no tensor memory; results carry the rounding of
                      every 16-deep partial sum (tolerance of GEMMTC.py:60-62).  0: fp32 */
    int raster_n;  /* 1: rasterisation groups are `raster` tile COLUMNS walked down M (a band of B stays in
                      L2 while A streams: for M > N); 0: `raster` tile rows walked along N.  cta_group = 1 */
} deca_gemm_cfg;

/* Host-only mirror of check_config (gemm_tir.py:101-120) for this tile space: shape limits,
 * N % 8 == 0 and K % 8 == 0 (16-byte row pitches), shared- and tensor-memory budgets. */
int deca_gemm16_check_config(int dtype, int64_t M, int64_t N, int64_t K, const deca_gemm_cfg *cfg);

/* The config deca_gemm16 uses when cfg == null, for a device with `sms` multiprocessors (host only;
 * the launch path passes the current device's count): 256x256x64 with 3 stages once such tiles give
 * every SM one or fill most of a wave, else the best-filling of 128x256, 128x128 and 128x64.  The Python operator's
 * default_config calls this function, so both routes to "the default" agree.
 * Takes the place of the defaults of GemmConfig (gemm_tir.py:42-76). */
int deca_gemm16_default_config(int64_t M, int64_t N, int64_t K, int sms, int acc_f16, deca_gemm_cfg *out);

/* Launches the GEMM.  A, B, C must be 16-byte aligned.  M, N, K need not be multiples of the
 * tile (partial tiles are zero-filled on load and clipped on store).  cfg == null selects
 * deca_gemm16_default_config for the current device.
 * Replaces runtime_mod["main"](a, b, c) of a GEMM kernel (RuntimeMod.py:204-208). */
int deca_gemm16(int dtype, const void *A, const void *B, void *C, int64_t M, int64_t N, int64_t K,
                const deca_gemm_cfg *cfg, void *stream);

/* Scratch memory deca_gemm16_ws needs for this problem and config on the current device
 * (0 when cfg->stream_k is 0 or splitting does not apply to the shape). */
int deca_gemm16_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K, const deca_gemm_cfg *cfg, size_t *bytes);

/* deca_gemm16 with caller-owned scratch memory, which the stream-K mode (cfg->stream_k = 1) uses
 * for the fp32 partial tiles of split output tiles and their ready flags.  `workspace` must be
 * 256-byte aligned, at least deca_gemm16_workspace_bytes long and ZERO on first use; a launch
 * that completes leaves the flags zero again, so the same workspace serves the next launch on
 * the same stream (launches that overlap in time need a workspace each).  After a non-zero
 * device status the workspace must be zeroed again.  The kernel is launched cooperatively in
 * this mode (the whole grid is resident).  Results differ from the unsplit kernel only by the
 * fp32 summation order of split tiles.  The reference has no split-k mode; this entry point
 * replaces the same runtime_mod["main"](a, b, c) call as deca_gemm16. */
int deca_gemm16_ws(int dtype, const void *A, const void *B, void *C, int64_t M, int64_t N, int64_t K,
                   const deca_gemm_cfg *cfg, void *workspace, size_t ws_bytes, void *stream);

/* deca_gemm16_ws on scratch memory built into the library: neither the caller nor the library
 * allocates anything.  The scratch is one file-scope device array of 20 MiB (flags + 160 fp32
 * tiles of up to 128 x 256), so the config must have stream_k = 1 and BM * BN <= 128 * 256, and
 * the device at most 160 SMs; a problem beyond that returns DECA_ERR_SCRATCH_LIMIT and launches
 * nothing.  The first call on a device looks the array's address up (with that device current):
 * make that call before any stream capture.  Every call on a device uses the same array, so calls
 * that overlap in time (two streams, two threads) race; calls on one stream are ordered and safe.
 * The array keeps what the last call left in it and is never cleared: each launch on a device is
 * numbered and a ready flag counts only when it holds the current launch's number, so flags left by
 * earlier launches (completed, or given up after a device timeout) cannot be taken for fresh ones.
 * No counterpart in the reference (it has no split-k mode and no library-owned buffers). */
int deca_gemm16_sk_static(int dtype, const void *A, const void *B, void *C, int64_t M, int64_t N, int64_t K,
                          const deca_gemm_cfg *cfg, void *stream);

/* M-sharded GEMM with the all-gather of the output fused into the epilogue: this rank computes
 * C_shard[M_shard, N] = A_shard[M_shard, K] @ B[K, N] and stores every output panel into rows
 * [rank * M_shard, (rank + 1) * M_shard) of EVERY rank's gathered output.  C_all[r] is the base of
 * rank r's [n_ranks * M_shard, N] buffer as addressable from this process (peer-mapped device
 * memory, e.g. symmetric memory or an opened IPC handle; C_all[rank] is this rank's own).  The
 * stores to peers are plain TMA stores over NVLink inside the GEMM kernel, no multicast.
 * 1 <= n_ranks <= 8; the config must stage panels in shared memory (epi_smem = 1).  The kernel
 * only writes: a reader of a gathered buffer must first synchronise with every writer (a barrier
 * across the ranks after the launches have completed).
 * No counterpart in the reference, whose GEMM is single-GPU; it serves the M-sharded
 * configuration (65536 x 8192 x 8192 over 8 GPUs) followed by an all-gather of C. */
int deca_gemm16_gather(int dtype, const void *A, const void *B, void *const *C_all, int n_ranks, int rank,
                       int64_t M_shard, int64_t N, int64_t K, const deca_gemm_cfg *cfg, void *stream);

/* ---------------------------------------------------------------------------------------
 * FlashAttention forward, fp16: O = softmax(scale * Q K^T [+ causal mask]) V with Q, K, V, O
 * contiguous [B, H, S, D], D = 64 or 128, fp32 softmax statistics.  The causal mask is
 * top-left aligned (key j visible to query i iff j <= i) and needs S_q == S_kv.
 * Replaces the kernel generated by make_flash_attn_fwd (src/kernels/flash_attn_tir.py:83-478);
 * the struct takes the place of FAConfig (flash_attn_tir.py:31-51).
 * ------------------------------------------------------------------------------------- */
typedef struct {
    int Br;      /* Q rows per tile: 128 (the tensor-memory lanes) */
    int Bc;      /* KV rows per pipeline step: 64 or 128 */
    int stages;  /* q_tiles = 1: depth of the K ring and of the V ring, 1..4;
                    q_tiles = 2: slots of the single ring K and V tiles share, 2..8
                    (must fit shared memory) */
    int q_tiles; /* Q tiles per CTA: 1, or 2 (two consecutive tiles share every K / V tile and
                    alternate on the tensor pipe; needs S_q % 256 == 0; Bc = 64 then needs p_tmem
                    and stages >= 4, and gives every tile two score buffers) */
    int p_tmem;  /* non-zero keeps P in tensor memory (the A operand of the P V product) instead of
                    staging it in shared memory */
    int persistent; /* 1: one CTA per SM walks a list of (head, Q-tile pair) items and overlaps the end of
                       one item with the start of the next; needs q_tiles = 2, Bc = 128, p_tmem; else 0 */
} deca_fa_cfg;

/* Host-only mirror of check_config (flash_attn_tir.py:70-80) for this tile space. */
int deca_fa_fwd_f16_check_config(int B, int H, int S_q, int S_kv, int D, int causal, const deca_fa_cfg *cfg);

/* Launches the kernel; all four tensors 16-byte aligned; cfg == null selects the library's default
 * for the shape (the persistent two-tile schedule when S_q % 256 == 0 and S_kv % 128 == 0).
 * Replaces runtime_mod["main"](q, k, v, o) (RuntimeMod.py:169-172). */
int deca_fa_fwd_f16(const void *Q, const void *K, const void *V, void *O, int B, int H, int S_q, int S_kv, int D,
                    float softmax_scale, int causal, const deca_fa_cfg *cfg, void *stream);

/* Head-sharded attention with the all-gather of the output fused into the epilogue: this rank
 * computes its [B, H, S_q, D] shard (B * H heads of the flattened batch x head axis) and stores
 * every output panel into heads [rank * B * H, (rank + 1) * B * H) of EVERY rank's gathered output.
 * O_all[r] is the base of rank r's [n_ranks * B * H, S_q, D] buffer as addressable from this
 * process (peer-mapped device memory; O_all[rank] is this rank's own).  Plain TMA stores over
 * NVLink inside the attention kernel, no multicast; 1 <= n_ranks <= 8.  The kernel only writes:
 * readers of a gathered buffer first synchronise with every writer.
 * No counterpart in the reference, whose kernels are single-GPU; it serves the head-sharded
 * configuration (B32 H32 S8192 D128 causal over 8 GPUs) followed by an all-gather of O. */
int deca_fa_fwd_f16_gather(const void *Q, const void *K, const void *V, void *const *O_all, int n_ranks, int rank,
                           int B, int H, int S_q, int S_kv, int D, float softmax_scale, int causal,
                           const deca_fa_cfg *cfg, void *stream);

/* ---------------------------------------------------------------------------------------
 * Residual addition + RMSNorm, the form RMSNorm takes between two layers:
 *   H = dt(h),  h = X + R in fp32;   y = h * rsqrt(mean(h^2) + eps) * W in fp32 (h is not rounded
 *   before it is normalised, and y is rounded once);   out = DECA_OUT_SAME: Y = dt(y), or
 *   out = DECA_OUT_E4M3: Y = e4m3(y / s), s = max |y| / 448 over the row (group = 0) or over each
 *   group of `group` (32, 64, 128 or 256) columns, the last one possibly short; scales[M, groups] fp32.
 *   A scale below the smallest normal fp32 number (all of the group's y zero, in practice) gives zeros.
 *   A NaN in a group makes its scale NaN.
 * Row strides in elements, at least N; W contiguous.  Any N: rows that are no multiple of 8 elements
 * or not 16-byte aligned take element-wise accesses.  H and Y (of DECA_OUT_SAME) may each be X or R itself (same
 * pointer and stride); other overlaps of an output are refused (DECA_ERR_UNSUPPORTED).  M = 0 launches nothing.
 * No counterpart in the reference, whose RMSNorm has neither residual nor 8-bit output.
 * ------------------------------------------------------------------------------------- */
enum { DECA_OUT_SAME = 0, DECA_OUT_E4M3 = 1 };
int deca_add_rmsnorm(int dtype, const void *X, int64_t x_stride, const void *R, int64_t r_stride, const void *W,
                     void *H, int64_t h_stride, void *Y, int64_t y_stride, float *scales, int64_t M, int64_t N,
                     float eps, int out, int group, void *stream);

/* ---------------------------------------------------------------------------------------
 * Rotary positions.  Pair i of a head's first rot_dim elements turns by the angle
 * 2 pi * position * turns[i] / 2^64:  (a, b) -> amplitude * (a cos - b sin, a sin + b cos).
 * DECA_ROT_HALF pairs (i, i + rot_dim / 2), DECA_ROT_INTERLEAVED pairs (2i, 2i + 1); elements from
 * rot_dim on are copied.  `turns` is a HOST array of rot_dim / 2 fixed-point fractions of a turn (it
 * travels with the launch), so angles are exact modulo a turn at any position; inverse = 1 turns the
 * other way, which is the transposed map, i.e. the gradient of the forward one.  fp32 arithmetic, one
 * rounding.  D and rot_dim even, 2 <= rot_dim <= D <= 256.
 * ------------------------------------------------------------------------------------- */
enum { DECA_ROT_HALF = 0, DECA_ROT_INTERLEAVED = 1 };
typedef struct {
    void *data;           /* device pointer to [tokens, heads, D], innermost dimension contiguous */
    int64_t token_stride; /* elements */
    int64_t head_stride;
} deca_tokens;
typedef struct {
    void *data; /* device pointer to [num_pages, page_size, H_kv, D], innermost dimension contiguous */
    int64_t page_stride; /* elements */
    int64_t row_stride;
    int64_t head_stride;
} deca_cache;
typedef struct {
    int D, rot_dim;
    int layout;            /* DECA_ROT_HALF or DECA_ROT_INTERLEAVED */
    int inverse;           /* 1: turn backwards */
    float amplitude;       /* factor on cos and sin (1 unless the scaling method asks for one) */
    const uint64_t *turns; /* host array, rot_dim / 2 entries */
} deca_rotation;

/* Y[t, h] = rotate(X[t, h], positions[t]); Y may be X itself (same pointer and strides), other overlaps of Y are
 * refused (DECA_ERR_UNSUPPORTED). */
int deca_rotary(int dtype, const deca_tokens *X, const deca_tokens *Y, const int32_t *positions, int64_t tokens,
                int heads, const deca_rotation *rot, void *stream);

/* Q_out = rotate(Q); row slots[t] of the cache = rotate(K[t]), V[t] in one launch, where slot s is row
 * s % page_size of page s / page_size.  A slot outside [0, num_pages * page_size) writes nothing (padding
 * rows carry -1); two tokens must not share a slot.  Q_out may be Q itself; other overlaps of Q_out and the caches with
 * each other or with an input are refused (DECA_ERR_UNSUPPORTED). */
int deca_rotary_append(int dtype, const deca_tokens *Q, const deca_tokens *K, const deca_tokens *V,
                       const deca_tokens *Q_out, const deca_cache *K_cache, const deca_cache *V_cache,
                       const int32_t *positions, const int64_t *slots, int64_t tokens, int H_q, int H_kv,
                       int64_t num_pages, int page_size, const deca_rotation *rot, void *stream);

/* ---------------------------------------------------------------------------------------
 * The bookkeeping of one serving step, on the device: from the cached length and the number of new
 * tokens of every request,
 *   cu_q[B + 1]   exclusive sum of new_lens;
 *   kv_lens[B]    ctx_lens + new_lens (at most table_width * page_size);
 *   block_table   entries ceil(ctx / page) .. ceil(kv / page) - 1 of every request take pages from the
 *                 free list: the i-th page that the step needs, in request order, is
 *                 free_pages[n_free - 1 - i] (-1 once the list is empty).  Other entries are left;
 *   n_free_out    what the list still holds;  short_out: pages that were missing (0: none);
 *   positions[T], slots[T]  of token t of the step: its place in its request, and
 *                 page * page_size + row of the cache (-1 where it has no page).  Entries behind the last
 *                 token get position 0 and slot -1; tokens beyond T are not written.
 * Negative lengths count as 0.  Outputs must not overlap the inputs or each other (DECA_ERR_UNSUPPORTED).
 * B <= 8192, page_size a power of two.
 * ------------------------------------------------------------------------------------- */
int deca_paged_step(const int32_t *ctx_lens, const int32_t *new_lens, int B, int32_t *block_table,
                    int64_t table_stride, int table_width, const int32_t *free_pages, int free_capacity,
                    const int32_t *n_free, int page_size, int64_t T, int32_t *cu_q, int32_t *kv_lens,
                    int32_t *positions, int64_t *slots, int32_t *n_free_out, int32_t *short_out, void *stream);

/* ---------------------------------------------------------------------------------------
 * Attention of new tokens over a paged cache: request r owns rows cu_q[r] .. cu_q[r + 1] - 1 of Q and O
 * and the first kv_lens[r] rows of the pages block_table[r][0 ..]; its new tokens are the last of them.
 * O[t, h] = softmax(scale * Q[t, h] K^T) V over the keys j <= kv_len - q_len + i (i = the token's place in
 * its request; causal = 0: over all kv_len keys), key head h / (H_q / H_kv).  A row that sees no key is
 * zero.  Rows of Q and O that belong to no request are not touched.  fp16 or bf16, fp32 scores, statistics
 * and accumulators; the probabilities are rounded to 16 bits for the product with V (their sum is not).  A NaN or an infinity in
 * what a row sees reaches it as in the formula (NaN for a NaN or a score of +inf, no weight for one of -inf); a row
 * whose scores are all -inf gives zeros.  D = 64 or 128, page_size 16, 32, 64, 128 or 256, H_q / H_kv <= 128.
 * Lengths are read on the device and clipped to what T and the table hold; a table entry that names no
 * page reads as zeros.  What a row cannot see never reaches it, whatever the cache holds there.
 * max_q / max_kv: upper bounds of a request's new tokens and cached length as the caller knows them;
 * they choose the schedule (any values give right results; a max_q far above a step's new tokens makes it up to twice as slow).  O may be Q (same pointer and strides); other overlaps of O
 * or the workspace with a buffer of the call are refused (DECA_ERR_UNSUPPORTED; _check leaves them to the launch).
 * Strides of Q, K and V are positive (K and V may have a head stride of 0: one key head seen as several).
 * ------------------------------------------------------------------------------------- */
typedef struct {
    int dtype;
    int B;               /* requests */
    int H_q, H_kv, D;
    int page_size;
    int causal;
    float scale;
    int64_t T;           /* rows of Q and O */
    int64_t num_pages;
    int64_t table_stride; /* elements */
    int table_width;
    int max_q, max_kv;
    deca_tokens Q, O;
    deca_cache K, V;
    const int32_t *block_table, *cu_q, *kv_lens;
    void *workspace;     /* deca_paged_attn_workspace_bytes (0: may be null), 256-byte aligned; contents need no
                            preparation.  Calls that overlap in time need one each */
    size_t workspace_bytes;
} deca_paged_attn_args;

int deca_paged_attn_check(const deca_paged_attn_args *a);
int deca_paged_attn_workspace_bytes(const deca_paged_attn_args *a, size_t *bytes);
int deca_paged_attn(const deca_paged_attn_args *a, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* DECA_B200_H */
