/*
 * enceladus_b200 — C ABI of the sm_100a kernel library (libenc_b200.so).
 *
 * This is the boundary a binding generator (ctypes, cffi, nanobind, cgo ...) binds.  It replaces, for
 * the kernel set, what the reference reaches through its generic Metal runtime:
 *   fr_stream_dispatch(stream, pso, name, plan, bufs, offsets, scalar_bytes, grid, tg)
 *                                                     src/enceladus/_C/enceladus_rt.h:137-139
 *   Stream.dispatch(...) in the nanobind module       src/enceladus/_C/bindings.mm:479-490
 *   CompiledKernel.launch(grid, values)               src/enceladus/runtime/launcher.py:457-512
 * The reference dispatches a JIT-compiled pipeline with an untyped binding plan; here every kernel of
 * the set is a typed entry point.  Conventions shared by all entry points:
 *
 *   - plain pointers and sizes only; every pointer is a DEVICE pointer on the current CUDA device
 *     unless the parameter name ends in `_host`;
 *   - the caller owns all buffers.  The library itself owns, per device: a 256-byte status block (bounded
 *     device-side waits report there) and the tile-descriptor scratch of enc_cumsum / enc_sum (see
 *     enc_cumsum); both are allocated on first use and freed at exit.  No other entry point allocates;
 *   - index arrays (lengths, positions, pages, tokens of the decoding step) are device data, so they are checked on the device:
 *     what they name out of range is skipped, and the next enc_synchronize on the device returns ENC_ERR_BAD_INDEX;
 *   - `stream` is a cudaStream_t / CUstream passed as void* (NULL = the legacy default stream); work
 *     is enqueued and the call returns without synchronising, like fr_stream_dispatch;
 *   - the return value is an enc_status; on failure enc_last_error() holds a message for the calling
 *     thread (the reference returns nonzero plus a message buffer, enceladus_rt.h:78-83,143-145);
 *   - sizes and strides are in ELEMENTS, 64-bit;
 *   - `variant` selects one of the hand-written tile variants of a kernel (0 .. enc_num_variants-1),
 *     or ENC_VARIANT_AUTO for the built-in choice; the autotuner iterates over them.
 */
#ifndef ENCELADUS_B200_H
#define ENCELADUS_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
    ENC_OK = 0,
    ENC_ERR_BAD_ARG = 1,      /* NULL pointer, negative size, unknown dtype/variant            */
    ENC_ERR_UNSUPPORTED = 2,  /* valid request this build has no kernel for                    */
    ENC_ERR_LAUNCH = 3,       /* CUDA reported an error at launch / in an earlier async launch */
    ENC_ERR_DEVICE_WAIT = 4,  /* a bounded device-side wait ran out (reported at sync)         */
    ENC_ERR_NO_MEMORY = 5,    /* scratch allocation failed                                     */
    ENC_ERR_BAD_INDEX = 6     /* an index array held a value out of range (reported at sync)   */
} enc_status;

typedef enum {
    ENC_F32 = 0,
    ENC_F16 = 1,
    ENC_BF16 = 2,
    ENC_I32 = 3,
    ENC_I8 = 4,
    ENC_I16 = 5,
    ENC_I64 = 6,
    ENC_U8 = 7
} enc_dtype;

typedef enum {
    ENC_K_SOFTMAX = 0,
    ENC_K_LAYERNORM = 1,
    ENC_K_RMSNORM = 2,
    ENC_K_GELU = 3,
    ENC_K_MATMUL = 4,
    ENC_K_ATTENTION = 5,
    ENC_K_HISTOGRAM = 6,
    ENC_K_CUMSUM = 7,
    ENC_K_ADD = 8,
    ENC_K_MATMUL_INT = 9,
    ENC_K_APPEND_KV = 10,
    ENC_K_PAGED_ATTENTION = 11,
    ENC_K_LOGITS = 12,
    ENC_K_COUNT = 13
} enc_kernel;

#define ENC_VARIANT_AUTO (-1)

/* ---- library / device -------------------------------------------------------------------- */

/* Message for the last failure on the calling thread ("" if none).  Replaces the `char *err`
 * out-parameters of fr_library_new / fr_stream_sync (enceladus_rt.h:78-83,143-145). */
const char *enc_last_error(void);

typedef struct {
    int device;               /* current CUDA device ordinal                         */
    int sm_count;             /* multiprocessors                                     */
    int cc_major, cc_minor;   /* compute capability                                  */
    int max_smem_per_block;   /* opt-in shared memory per block, bytes               */
    int l2_bytes;
    uint64_t global_mem;      /* bytes                                               */
    char name[128];
} enc_device_info_t;

/* Replaces fr_device_query / fr_device_name (enceladus_rt.h:29-33). */
int enc_device_info(enc_device_info_t *out);

/* Number of hand-written tile variants of a kernel, and a one-line description of one
 * ("rows_per_cta=8 threads_per_row=32", "tile=128x256x64 stages=4", ...).  The autotuner uses
 * these in place of the reference's (BM, BN, BK, num_warps) config lists (src/enceladus/configs.py:19-44). */
int enc_num_variants(int kernel);
int enc_variant_info(int kernel, int variant, char *out, size_t n);

/* Waits for `stream` and reports errors of earlier asynchronous launches, including a bounded
 * device-side wait that ran out (ENC_ERR_DEVICE_WAIT).  Replaces fr_stream_sync (enceladus_rt.h:143-145). */
int enc_synchronize(void *stream);

/* ---- bandwidth-bound kernels -------------------------------------------------------------- */

/* Row softmax over the last axis, float32 math, output in the input dtype.
 * Replaces softmax_kernel[(rows,)](out, in, stride_in, stride_out, n_cols, BLOCK)   examples/02_softmax.py:15-38
 * dtype: ENC_F32 | ENC_F16 | ENC_BF16.  Rows may be strided; elements of a row are contiguous. */
int enc_softmax(const void *in, void *out, int64_t rows, int64_t cols, int64_t stride_in,
                int64_t stride_out, int dtype, int variant, void *stream);

/* LayerNorm forward: y = (x-mean)*rstd*w + b, mean/rstd float32 per row (biased variance: one pass of sum and
 * sum of squares, the centred second pass of the reference for rows with mean^2 > 16 var).
 * Replaces layernorm_kernel[(rows,)](x, y, w, b, mean, rstd, stride_x, stride_y, n_cols, eps, BLOCK)
 *                                                                                    examples/03_layernorm.py:15-57
 * x, y, w, b share `dtype`.  mean / rstd may be NULL (not written). */
int enc_layernorm(const void *x, void *y, const void *w, const void *b, float *mean, float *rstd,
                  int64_t rows, int64_t cols, int64_t stride_x, int64_t stride_y, float eps,
                  int dtype, int variant, void *stream);

/* RMSNorm forward: y = x * (1/sqrt(mean(x^2)+eps)) * w.
 * Replaces rmsnorm_kernel[(rows,)](x, w, out, stride_x, stride_out, n_cols, eps, BLOCK)  examples/06_rmsnorm.py:15-37 */
int enc_rmsnorm(const void *x, const void *w, void *y, int64_t rows, int64_t cols,
                int64_t stride_x, int64_t stride_y, float eps, int dtype, int variant, void *stream);

/* Fused elementwise GELU: t = x*scale + bias[i % n_cols]; out = gelu(t).
 * mode 0 = erf form (0.5*t*(1+erf(t*0.70710677f))), mode 1 = tanh form
 * (0.5*t*(1+tanh(0.7978846f*(t+0.044715f*t^3)))).  bias may be NULL (then no bias is added and
 * n_cols is ignored); scale is applied only when has_scale != 0.
 * Replaces fused_gelu_kernel[(cdiv(n,BLOCK),)](x, bias, out, n, n_cols, scale, BLOCK)    examples/05_fused_gelu.py:17-33 */
int enc_gelu(const void *x, const void *bias, void *out, int64_t n, int64_t n_cols, float scale,
             int has_scale, int mode, int dtype, int variant, void *stream);

/* out = x + y.  Replaces add_kernel  examples/01_vector_add.py:15-22 */
int enc_add(const void *x, const void *y, void *out, int64_t n, int dtype, int variant, void *stream);

/* ---- integer kernels ---------------------------------------------------------------------- */

/* hist[b] += #{ i : floor((float(x[i]) - lo) * inv_width) == b, 0 <= b < num_bins }, int32 counts.
 * `hist` is accumulated into (the caller zero-fills it, as enceladus.new_zeros does).
 * Replaces histogram_kernel[(cdiv(n,BLOCK),)](x, hist, n, lo, inv_width, NUM_BINS, BLOCK)  examples/09_histogram.py:17-34
 * dtype: ENC_F32 | ENC_F16 | ENC_BF16 | ENC_I32. */
int enc_histogram(const void *x, int32_t *hist, int64_t n, float lo, float inv_width,
                  int64_t num_bins, int dtype, int variant, void *stream);

/* Inclusive scan along rows: out[r, c] = sum_{c' <= c} in[r, c'] (or c' >= c when reverse != 0).
 * Integers narrower than 32 bits accumulate and are written as int32; int32 wraps modulo 2^32;
 * float16/bfloat16 accumulate in float32 and are rounded on store; out dtype = enc_cumsum_out_dtype.
 * rows == 1 is the flat form (any length, single-pass decoupled look-back over tiles).
 * `seed` (device pointer to ONE accumulator-typed value, or NULL) is added to every output of the
 * flat form: the exclusive offset of this shard when one array is split across GPUs.
 * Scratch: the flat form keeps 8 bytes per 4096-element tile plus a 64-byte header in a per-device
 * buffer the library allocates on first use and grows on demand (cudaMalloc; freed at exit).
 * Replaces cumsum_kernel[(cdiv(rows,BLOCK_M),)](out, in, n_rows, n_cols, stride_in, stride_out, REVERSE, ...)
 *                                                                                    examples/10_cumsum.py:17-42 */
int enc_cumsum(const void *in, void *out, int64_t rows, int64_t cols, int64_t stride_in,
               int64_t stride_out, int reverse, int dtype, const void *seed, int variant,
               void *stream);
int enc_cumsum_out_dtype(int dtype);

/* The flat form of enc_cumsum (rows == 1, forward) for callers that must not allocate device memory:
 * a framework that owns the whole device through its own pool, a serving loop that cannot take the
 * device-wide stall of an allocation, code under a "nothing is allocated after start-up" rule.  This
 * entry point has no counterpart in the reference.  It calls no cudaMalloc/cudaFree or other allocating
 * routine; the look-back descriptors live in a 1 MiB array inside the library image (held by every GPU
 * that loads the library until the process exits), which limits n to 2^30 elements — longer inputs are
 * refused with ENC_ERR_UNSUPPORTED.  The first call on a device resolves the array's device address;
 * make that call before any stream capture.  Every call on a device shares the array: calls on one
 * stream are safe, calls that overlap on the GPU race.  `status` (device pointer owned by the caller, or
 * NULL) is set non-zero if a bounded device-side wait ran out, in which case the output is invalid.  With
 * status == NULL that timeout is recorded only in a spare word of the array that nothing reads, so the
 * failure is SILENT (enc_synchronize does not report it either): pass a status word unless a wrong output
 * would be caught downstream.  Same dtypes and results as enc_cumsum except ENC_I64. */
int enc_cumsum_noalloc(const void *in, void *out, int64_t n, int dtype, const void *seed,
                       unsigned *status, void *stream);

/* total[0] = sum of n elements in the accumulator type of enc_cumsum (int32 wrap / float32).
 * Pass 1 of the multi-GPU flat scan (local total -> all-gather -> seed).  No counterpart in the
 * reference, which has no multi-device path. */
int enc_sum(const void *in, void *total, int64_t n, int dtype, void *stream);

/* offset[0] = totals[0] + ... + totals[index-1] (0 for index 0) in the accumulator type of enc_cumsum for
 * `dtype` (32-bit wrap, float32 or int64 adds in shard order): the `seed` of shard `index` once the per-shard
 * totals of enc_sum have been all-gathered into `totals` (device, `count` values).  A one-thread kernel on
 * `stream`, so that the two passes of the multi-GPU scan and the collective between them stay stream-ordered
 * with no host round trip.  No counterpart in the reference (single device). */
int enc_scan_offset(const void *totals, int count, int index, void *offset, int dtype, void *stream);

/* ---- tensor-core kernels ------------------------------------------------------------------ */

/* C = epilogue(A @ B): A [M,K] (lda), B [K,N] (ldb), C [M,N] (ldc), all row-major with unit inner
 * stride, float32 accumulation on tcgen05 tensor cores (float32 operands: CUDA cores), C in the operand dtype.
 * epilogue 0: identity.  epilogue 1: t = acc + bias[n]; 0.5*t*(1+erf(t*0.70710677f)).
 * Out-of-range tile elements read as zero and are not stored (descriptor semantics,
 * src/enceladus/language/ops.py:495-514).  dtype: ENC_F16 | ENC_BF16 | ENC_F32.  Operands need no alignment:
 * 16-byte aligned bases and leading dimensions that are multiples of 8 are fetched by TMA, anything else (the
 * reference's 513^3 shape, benchmarks/bench_matmul.py:30) by loader warps inside the same tensor-core kernel;
 * nothing is copied or allocated.
 * Replaces matmul_bias_gelu_kernel[(cdiv(N,BN),cdiv(M,BM))](a, b, bias, c, M, N, K, lda, ldb, ldc, BM, BN, BK)
 *                                                                                    examples/07_matmul_fused.py:17-48
 * and matmul_desc_kernel                                                             examples/04_matmul.py:21-63 */
int enc_matmul(const void *a, const void *b, const void *bias, void *c, int64_t M, int64_t N,
               int64_t K, int64_t lda, int64_t ldb, int64_t ldc, int epilogue, int dtype,
               int variant, void *stream);

/* C = A @ B for integer operands: A [M,K] (lda), B [K,N] (ldb), both of `dtype`, C [M,N] int32 (ldc), row-major
 * with unit inner stride.  int32 accumulation, exact: products and sums wrap modulo 2^32
 * (integer tl.dot, src/enceladus/language/ops.py:1255-1259).  ENC_I8 and ENC_U8 run on the tcgen05 tensor cores
 * (kind::i8) when A and B are 16-byte aligned with leading dimensions that are multiples of 16, otherwise and for
 * ENC_I16 / ENC_I32 on CUDA cores.  Out-of-range tile elements read as zero and are not stored.
 * Replaces int8_matmul_kernel[(cdiv(N,BN),cdiv(M,BM))](a, b, c, M, N, K, BM, BN, BK)   benchmarks/bench_matmul.py:100-131
 * and the integer tl.dot kernels of                                                   tests/test_interpreter.py:808-835 */
int enc_matmul_int(const void *a, const void *b, void *c, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                   int64_t ldc, int dtype, int variant, void *stream);

/* Flash-attention forward over `bh` independent (batch, head) slices of shape [seq, head_dim]:
 * O = softmax(Q K^T * sm_scale [causal]) V, base-2 online softmax in float32, P rounded to the input
 * dtype before P@V, O in the input dtype.  lse (float32 [bh, seq], may be NULL) receives
 * ln2*(m + log2 l) of the running statistics.  stride_h = elements between slices, stride_m =
 * elements between rows (head_dim contiguous).  dtype: ENC_F16 | ENC_BF16 | ENC_F32; head_dim <= 128.
 * float16 / bfloat16 with head_dim 64 or 128, 16-byte aligned tensors and strides that are multiples of 8
 * run on the tcgen05 tensor cores; every other accepted shape runs on a CUDA-core kernel with the same
 * arithmetic.
 * Replaces attention_kernel[(cdiv(S,BLOCK_M), B*H)](q, k, v, o, sm_scale, N_CTX, stride_h, stride_m, HEAD_DIM, ...)
 *                                                                                    examples/08_flash_attention.py:30-103 */
int enc_attention_fwd(const void *q, const void *k, const void *v, void *o, float *lse, int64_t bh,
                      int64_t seq, int64_t head_dim, int64_t stride_h, int64_t stride_m,
                      float sm_scale, int causal, int dtype, int variant, void *stream);

/* ---- decoding step -------------------------------------------------------------------------- */

/* A paged key-value cache.  k and v are pools of num_pages pages; a page holds page_size tokens of kv_heads heads
 * of head_dim elements.  Any layout with contiguous head elements is described by its strides (page-head-token-dim
 * and page-token-head-dim alike), k and v each with their own.  block_table[s * stride_table + i] is the page that holds
 * tokens i*page_size .. (i+1)*page_size-1 of sequence s.  Several sequences may name the same page (a shared prefix). */
typedef struct {
    void *k, *v;
    const int32_t *block_table; /* [num_seqs, table_width]                        */
    int64_t num_pages, page_size, kv_heads, head_dim;
    int64_t num_seqs, table_width, stride_table;
    int64_t k_stride_page, k_stride_head, k_stride_token;
    int64_t v_stride_page, v_stride_head, v_stride_token;
} enc_paged_cache;

/* Appends one key and one value per token to the cache and rotates queries and keys by their positions on the way.
 * Token t belongs to sequence seq_ids[t] and has position positions[t] in it; seq_ids[t] < 0 marks padding: nothing is
 * written for that token.  Of every query and key head the first rot_dim elements turn in pairs,
 *   a' = a*cos - b*sin,  b' = b*cos + a*sin,   (a, b) = elements (i, i + rot_dim/2), or (2i, 2i+1) when `interleaved`,
 * in float32 with one rounding, by cos / sin [num_positions, rot_dim/2] (float32, rows stride_cos apart) at the token's
 * position; the other elements and the values are copied.  q and q_out may be NULL (no queries) or the same tensor;
 * rot_dim 0 (cos and sin then unused) appends without rotation.
 * k, v: [tokens, kv_heads, head_dim], q, q_out: [tokens, q_heads, head_dim], strides per token and head, elements of a
 * head contiguous.  All share `dtype` (ENC_F32 | ENC_F16 | ENC_BF16) with the cache.
 * A token whose sequence, position or page is out of range is skipped and enc_synchronize returns ENC_ERR_BAD_INDEX.
 * Two tokens of one call must not name the same place in the cache: which of them stays there is not defined.
 * No counterpart in the reference, whose attention (examples/08_flash_attention.py:30-103) has no cache. */
typedef struct {
    const void *k, *v, *q;
    void *q_out;
    const float *cos, *sin;
    const int32_t *seq_ids, *positions;
    int64_t tokens, q_heads, rot_dim, interleaved, num_positions;
    int64_t k_stride_token, k_stride_head, v_stride_token, v_stride_head;
    int64_t q_stride_token, q_stride_head, o_stride_token, o_stride_head, stride_cos;
} enc_append_args;
int enc_append_kv(const enc_paged_cache *cache, const enc_append_args *args, int dtype, int variant, void *stream);

/* Attention of one new token per sequence over the cache: for every sequence s < cache->num_seqs and query head h,
 * o[s, h] = softmax(q[s, h] . K^T * sm_scale) V over the first seq_lens[s] tokens of the sequence (the last `window` of
 * them when window > 0), with head h reading kv head h / (q_heads / kv_heads).  Statistics and sums in float32.  A row
 * without keys (length zero), or whose weights sum to zero, is zero with lse -inf.  lse: float32 [num_seqs, q_heads] or
 * NULL.  Cache contents past a sequence's length or in front of its window are never used.
 * q, o: [num_seqs, q_heads, head_dim] with strides per sequence and head; all of `dtype`; head_dim <= 256.  o may be q
 * itself: a row's queries are read by the CTAs that write it, or before the launch that joins its pieces.
 * The keys of all sequences and heads are dealt out evenly over the GPU, whatever their lengths: the schedule is computed
 * on the device from seq_lens, so a captured launch follows the lengths it finds.  Pieces that do not finish a row go
 * through `work`, a buffer of at least enc_paged_attention_work_bytes() bytes, 16-byte aligned, whose contents need
 * no preparation and mean nothing afterwards; launches that may overlap need buffers of their own.
 * A length or page out of range is cut or skipped and enc_synchronize returns ENC_ERR_BAD_INDEX.
 * Counterpart in the reference for a whole sequence without a cache: examples/08_flash_attention.py:30-103 */
typedef struct {
    const void *q;
    void *o;
    float *lse;
    const int32_t *seq_lens;
    void *work;
    int64_t work_bytes, q_heads, q_stride_seq, q_stride_head, o_stride_seq, o_stride_head, window;
    double sm_scale;
} enc_paged_attention_args;
int enc_paged_attention(const enc_paged_cache *cache, const enc_paged_attention_args *args, int dtype, int variant, void *stream);
/* Bytes of `work` that enc_paged_attention needs at most for caches and tables of these sizes (pointers and strides are not
 * looked at) on the current device, 0: none; -1 on a bad argument. */
int64_t enc_paged_attention_work_bytes(const enc_paged_cache *cache, int64_t q_heads, int dtype, int variant);

/* Penalties, biases and grammar masks on logits [rows, vocab], one pass, float32 arithmetic, output in `dtype`:
 *   x = logits[r, t]
 *   t among tokens[r, :lens[r]]                         : x = x > 0 ? x / repetition[r] : x * repetition[r]
 *   t n > 0 times in tokens[r, prompt_lens[r]:lens[r]]  : x = x - (frequency[r] * n + presence[r])
 *   x = x + (sum of bias_values[r, i] with bias_ids[r, i] == t, in order of i)
 *   bit t % 32 of mask[r, t / 32] clear                 : x = -inf
 * tokens (int32 [rows, .], rows stride_tokens apart, `history` columns), lens, prompt_lens, repetition, frequency and
 * presence come together or are all NULL; bias_ids / bias_values [rows, num_biases] (an id of -1 is an unused place) and
 * mask [rows, stride_mask words] each may be NULL.  out may be logits itself.  Masked logits are -inf whatever they were.
 * A token, id or length out of range is ignored or cut and enc_synchronize returns ENC_ERR_BAD_INDEX.
 * No counterpart in the reference; the rows continue in softmax_kernel, examples/02_softmax.py:15-38 */
typedef struct {
    const void *logits;
    void *out;
    const int32_t *tokens, *lens, *prompt_lens;
    const float *repetition, *frequency, *presence;
    const int32_t *bias_ids;
    const float *bias_values;
    const int32_t *mask;
    int64_t rows, vocab, stride_in, stride_out, history, stride_tokens, num_biases, stride_bias, stride_mask;
} enc_logits_args;
int enc_penalize_logits(const enc_logits_args *args, int dtype, int variant, void *stream);

/* ---- test hook ---------------------------------------------------------------------------- */

/* Forces the NEXT entry-point call on this thread to return `status` without launching anything
 * (host-side failure injection for the binding's error path; the reference injects failures with a
 * proxy around its native stream, tests/test_runtime.py:460-514).  0 clears it. */
void enc_test_fail_next(int status);

/* Launches one thread that polls a flag nothing sets, `polls` times at most (1 us apart, polls <=
 * 1000000), then gives up exactly as the library's bounded device-side waits do: it raises the device
 * status word and returns, so the next enc_synchronize reports ENC_ERR_DEVICE_WAIT and the context stays
 * usable.  Exercises the timeout path without hanging or faulting the GPU (the reference tests its
 * lost-sentinel timeout the same way, with a bounded wait: src/enceladus/runtime/stream.py:153-168). */
int enc_test_device_wait(unsigned int polls, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ENCELADUS_B200_H */
