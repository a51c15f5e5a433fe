/*
 * qdl_flash_born.h -- C ABI of the MI355X (gfx950) flash-Born attention library
 * (libqdl_flash_born.so).
 *
 * Born attention, per (b, h):
 *   a_ij = max(0, scale_h * q_i . k_j) * M_ij,  p_ij = a_ij^2,
 *   Z_i  = sum_j p_ij + eps,                    O_i  = sum_j p_ij v_j / Z_i,
 *   M_ij = [causal => j <= i] & [window > 0 => i - j < window] & [doc_i == doc_j].
 *
 * Conventions shared by every entry point:
 *   - q, k, v, out, dout, dq, dk, dv: contiguous (B, H, T, D) arrays of the
 *     element type `dtype`, base addresses 16-byte aligned.
 *   - z, delta: contiguous (B, H, T) fp32.
 *   - scale: `n_scale` fp32 values in device memory, n_scale == 1 (shared) or
 *     n_scale == H (per head, indexed by h).
 *   - doc_ids: contiguous (B, T) int32 in device memory, or NULL.
 *   - D must be a multiple of 8 in [8, 256].  (The Python host zero-pads other
 *     head dims up to the next multiple of 8; padding is exact.)
 *   - Every call is asynchronous on `stream` (a hipStream_t; NULL is the null
 *     stream), allocates nothing and keeps no state between calls.  The caller
 *     owns all buffers, including the workspace.
 *   - Return value: 0 on success; a negative QDL_BORN_E_* code for invalid
 *     arguments (nothing was launched); a positive hipError_t value when a
 *     launch failed.  qdl_flash_born_strerror() describes any code.
 */
#ifndef QDL_FLASH_BORN_H
#define QDL_FLASH_BORN_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types (the compute dtype of the reference's autograd Function). */
#define QDL_BORN_DTYPE_F32 0
#define QDL_BORN_DTYPE_F16 1
#define QDL_BORN_DTYPE_BF16 2

/* Error codes (negative: rejected before any launch). */
#define QDL_BORN_OK 0
#define QDL_BORN_E_DTYPE (-1)
#define QDL_BORN_E_SHAPE (-2)
#define QDL_BORN_E_HEADDIM (-3)
#define QDL_BORN_E_ALIGN (-4)
#define QDL_BORN_E_NULL (-5)
#define QDL_BORN_E_SCALE (-6)
#define QDL_BORN_E_WINDOW (-7)
#define QDL_BORN_E_WORKSPACE (-8)
#define QDL_BORN_E_TAU (-9)
#define QDL_BORN_E_TABLE (-10)
#define QDL_BORN_E_ROPEDIM (-11)
#define QDL_BORN_E_SCRATCH (-12)
#define QDL_BORN_E_HEADS (-13)
#define QDL_BORN_E_STRIDE (-14)
#define QDL_BORN_E_PAGE (-15)
#define QDL_BORN_E_BUDGET (-16)

/* Size of the fixed device array qdl_flash_born_bwd_noalloc takes its
 * workspace from (one per GPU): 16 MiB, enough for B * H * T up to about
 * 1.39 million rows (C5's B16 H16 T2048 needs 6.3 MB). */
#define QDL_BORN_BWD_SCRATCH_BYTES (16 * 1024 * 1024)

typedef struct ihipStream_t *qdl_stream_t; /* == hipStream_t */

/* Library version string, e.g. "qdl_flash_born 0.1.0 gfx950". */
const char *qdl_flash_born_version(void);

/* Human-readable text for a return code of any entry point. */
const char *qdl_flash_born_strerror(int code);

/* 1 if (dtype, head_dim) is served by the kernels without host padding. */
int qdl_flash_born_supported(int dtype, int64_t head_dim);

/*
 * Forward pass.  Writes out (B, H, T, D) and z (B, H, T) = sum_j p_ij + eps.
 *
 * Replaces the launch of `_flash_born_fwd_kernel[grid](...)` in
 * `_FlashBornAttentionFn.forward` (Vengo/QuantumDLBlocks
 * src/qdlblocks/kernels/flash_born.py:475-513); arguments carry the same
 * meaning as that launch's (pointers, B/H/T/D, PER_HEAD_SCALE via n_scale,
 * IS_CAUSAL, WINDOW_SIZE, HAS_DOC_IDS via doc_ids != NULL, EPS).
 */
int qdl_flash_born_fwd(int dtype, int64_t B, int64_t H, int64_t T, int64_t D,
                       const void *q, const void *k, const void *v, void *out,
                       float *z, const float *scale, int64_t n_scale,
                       const int32_t *doc_ids, int is_causal,
                       int64_t window_size, double eps, qdl_stream_t stream);

/* Bytes of device workspace qdl_flash_born_bwd needs for this problem. */
int64_t qdl_flash_born_bwd_workspace_size(int dtype, int64_t B, int64_t H,
                                          int64_t T, int64_t D,
                                          int64_t n_scale);

/*
 * Backward pass.  Given the forward's out and z and the upstream gradient
 * dout, writes dq, dk, dv (B, H, T, D) and dscale (n_scale fp32 values:
 * per-head sums, or the total when n_scale == 1).  The dscale reduction is
 * deterministic (fixed-order, no atomics).
 *
 * Replaces the two launches `_flash_born_bwd_kernel[grid_n](...)` and
 * `_flash_born_bwd_dq_kernel[grid_m](...)` in `_FlashBornAttentionFn.backward`
 * (flash_born.py:554-612) together with the zero-initialised dscale buffer
 * they accumulate into (flash_born.py:536).
 */
int qdl_flash_born_bwd(int dtype, int64_t B, int64_t H, int64_t T, int64_t D,
                       const void *q, const void *k, const void *v,
                       const void *out, const void *dout, const float *z,
                       const float *scale, int64_t n_scale,
                       const int32_t *doc_ids, int is_causal,
                       int64_t window_size, double eps, void *dq, void *dk,
                       void *dv, float *dscale, void *workspace,
                       int64_t workspace_bytes, qdl_stream_t stream);

/*
 * Backward pass that allocates nothing: qdl_flash_born_bwd with the
 * workspace taken from a fixed device array of QDL_BORN_BWD_SCRATCH_BYTES
 * inside the library instead of from the caller.
 *
 * No counterpart in the reference: it is for callers that cannot allocate
 * device memory (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc).  It calls no hipMalloc, hipFree or allocating
 * library routine; the caller still passes every input and output.  Each GPU
 * holds its own array until the process ends; its device address is looked
 * up on the first call on that GPU, so call with the device of `stream`
 * current.  Every call on one GPU shares that GPU's array: calls that overlap
 * on one GPU (other streams or threads) race.  A problem whose workspace
 * (qdl_flash_born_bwd_workspace_size) exceeds QDL_BORN_BWD_SCRATCH_BYTES is
 * rejected with QDL_BORN_E_SCRATCH before any HIP call; otherwise arguments,
 * results and return codes are those of qdl_flash_born_bwd.
 */
int qdl_flash_born_bwd_noalloc(int dtype, int64_t B, int64_t H, int64_t T,
                               int64_t D, const void *q, const void *k,
                               const void *v, const void *out,
                               const void *dout, const float *z,
                               const float *scale, int64_t n_scale,
                               const int32_t *doc_ids, int is_causal,
                               int64_t window_size, double eps, void *dq,
                               void *dk, void *dv, float *dscale,
                               qdl_stream_t stream);

/*
 * Purified-Born attention (flash_born.py:693-1341): weights
 *   p_ij = relu(scale_h (q_i.k_j - tau_h))^4 + eps_base relu(q_i.k_j)^2
 * under the same masks, Z_i = sum_j p_ij + eps, O_i = sum_j p_ij v_j / Z_i.
 * `tau` holds n_tau fp32 values in device memory (1 or H, like scale).  The
 * output is fp32 whatever the input dtype, as the reference's kernel writes
 * an fp32 output (flash_born.py:1102) that its autograd function then casts.
 */

/* Forward: writes out (B, H, T, D) fp32 and z (B, H, T) fp32.
 * Replaces the launch of `_flash_purified_born_fwd_kernel[grid](...)` in
 * `_FlashPurifiedBornAttentionFn.forward` (flash_born.py:1110-1151). */
int qdl_flash_purified_born_fwd(int dtype, int64_t B, int64_t H, int64_t T,
                                int64_t D, const void *q, const void *k,
                                const void *v, float *out, float *z,
                                const float *scale, int64_t n_scale,
                                const float *tau, int64_t n_tau,
                                double eps_base, const int32_t *doc_ids,
                                int is_causal, int64_t window_size,
                                double eps, qdl_stream_t stream);

/* Bytes of device workspace qdl_flash_purified_born_bwd needs. */
int64_t qdl_flash_purified_born_bwd_workspace_size(int dtype, int64_t B,
                                                   int64_t H, int64_t T,
                                                   int64_t D);

/* Backward: given the forward's fp32 out and z and the upstream gradient dout
 * (input dtype), writes dq, dk, dv (input dtype), dscale (n_scale fp32) and
 * dtau (n_tau fp32), both reduced in a fixed order (deterministic).
 * Replaces the two launches `_flash_purified_born_bwd_kernel[grid_n](...)`
 * and `_flash_purified_born_bwd_dq_kernel[grid_m](...)` in
 * `_FlashPurifiedBornAttentionFn.backward` (flash_born.py:1197-1262) with
 * the zero-initialised dscale / dtau buffers they accumulate into
 * (flash_born.py:1178-1179). */
int qdl_flash_purified_born_bwd(int dtype, int64_t B, int64_t H, int64_t T,
                                int64_t D, const void *q, const void *k,
                                const void *v, const float *out,
                                const void *dout, const float *z,
                                const float *scale, int64_t n_scale,
                                const float *tau, int64_t n_tau,
                                double eps_base, const int32_t *doc_ids,
                                int is_causal, int64_t window_size, void *dq,
                                void *dk, void *dv, float *dscale, float *dtau,
                                void *workspace, int64_t workspace_bytes,
                                qdl_stream_t stream);

/*
 * Struct form of the forward and backward, for hosts that call often: one
 * argument block (every field 8 bytes, so it can be packed from a script) in
 * place of 17 to 26 arguments, and
 *   - scale == NULL takes scale_value for every head (likewise tau), so a
 *     plain number needs no device copy and no synchronisation;
 *   - dscale / dtau == NULL: that gradient is not wanted, and the launches
 *     that reduce it are left out;
 *   - purified != 0 selects the purified weights (out is then fp32; out16 takes
 *     the output rounded to the element type), prologue
 *     != 0 the fused Q/K prologue (Born forward).
 * param_grads keeps fp32 and fp16 purified calls whose scale or tau is trained
 * on the kernels of the positional entry points: dscale is a cancelling sum,
 * which the output's last bits (another summation order) move by up to 4e-3.
 * Other fields, results and return codes are those of the positional entry
 * points; struct_bytes must be sizeof(qdl_born_call) (else QDL_BORN_E_SHAPE).
 * Unused fields are ignored.
 */
typedef struct qdl_born_call {
    int64_t struct_bytes;
    int64_t dtype, B, H, T, D;
    const void *q, *k, *v;
    void *out; /* written by the forward, read by the backward */
    float *z;
    const float *scale;
    int64_t n_scale;
    double scale_value;
    const int32_t *doc_ids;
    int64_t is_causal, window_size;
    double eps;
    int64_t purified;
    const float *tau;
    int64_t n_tau;
    double tau_value;
    double eps_base;
    void *out16;         /* purified forward, 16-bit: the output in the element type (out may then be NULL: no backward) */
    int64_t param_grads; /* purified forward: != 0 if the backward will be asked for dscale or dtau */
    /* backward */
    const void *dout;
    void *dq, *dk, *dv;
    float *dscale, *dtau;
    void *workspace; /* the positional entry points' size functions */
    int64_t workspace_bytes;
    /* forward of the fused Q/K prologue (qdl_flash_born_fwd_qk_prologue) */
    int64_t prologue; /* != 0: q, k are raw rows, the fields below apply */
    int64_t q_strides[3], k_strides[3];
    const float *cos_table, *sin_table;
    int64_t n_freq, table_ld;
    double norm_eps;
    void *q_out, *k_out;
    float *q_rinv, *k_rinv;
} qdl_born_call;

int qdl_flash_born_forward_call(const qdl_born_call *call, qdl_stream_t stream);
int qdl_flash_born_backward_call(const qdl_born_call *call, qdl_stream_t stream);

/*
 * Q/K prologue of SubspaceProjectorBornAttention.forward (attention.py:573-589,
 * without the optional wave filter and partial key offset), fused into one
 * pass per tensor:
 *   x' = l2_normalize(apply_unitary_rope(x, c, s), eps)       for x in {q, k}
 * with apply_unitary_rope (functional.py:104-121) rotating column pairs
 * (i, i + D/2):  y_i = x_i c_ti - x_{i+D/2} s_ti,  y_{i+D/2} = x_i s_ti + x_{i+D/2} c_ti,
 * and l2_normalize (functional.py:36-80): x' = y / sqrt(sum y^2 + eps), the
 * sum in fp32.  For 16-bit dtypes every product, sum and c, s themselves are
 * rounded to the dtype as the reference's tensor ops round them; the norm is
 * formed in fp32 from the rounded y.
 *
 * Row tensors (q, k, dq, dk) are (B, H, T, D) with element strides
 * strides[0..2] for b, h, t and unit stride along D, so the (B, T, H, D)
 * output of a Q/K projection is passed without a transposing copy.  q_out,
 * k_out, dq_out, dk_out are contiguous (B, H, T, D); q_rinv, k_rinv are
 * contiguous (B, H, T) fp32 holding 1 / sqrt(sum y^2 + eps) per row.
 * cos_table, sin_table: fp32, row t (t = 0 .. T-1) at t * table_ld; column
 * i < n_freq holds the angle table for pair i; pairs i >= n_freq are rotated
 * by angle 0 (cos 1, sin 0), the reference's padding of short tables
 * (attention.py:574-582).  cos_table == NULL skips the rotation.
 * Either tensor may be left out by passing NULL for all of its pointers;
 * q_rinv, k_rinv may be NULL on their own (1/norm is then not written: no
 * backward follows).  D must be even, 2 <= D <= 256.
 */

/* Forward.  Replaces the apply_unitary_rope and l2_normalize calls on Q and K
 * at attention.py:583-589 (and the .contiguous() copies at attention.py:516-517
 * when the projection output is passed strided). */
int qdl_flash_born_qk_prologue_fwd(int dtype, int64_t B, int64_t H, int64_t T,
                                   int64_t D, const void *q,
                                   const int64_t *q_strides, const void *k,
                                   const int64_t *k_strides,
                                   const float *cos_table,
                                   const float *sin_table, int64_t n_freq,
                                   int64_t table_ld, double eps, void *q_out,
                                   void *k_out, float *q_rinv, float *k_rinv,
                                   qdl_stream_t stream);

/* Backward: given the gradients dq_out, dk_out of q_out, k_out, the forward's
 * outputs and q_rinv, k_rinv, writes dq, dk (strided like the forward's
 * inputs):  g = (dx' - (dx'.x') x') rinv  (functional.py:50-57, rounded to
 * the dtype), then the transposed rotation  dx_i = g_i c + g_{i+D/2} s,
 * dx_{i+D/2} = g_{i+D/2} c - g_i s, each product and sum rounded to the dtype
 * as autograd's bf16 / fp16 ops round them.  Replaces the autograd backward of
 * the calls at attention.py:583-589. */
int qdl_flash_born_qk_prologue_bwd(int dtype, int64_t B, int64_t H, int64_t T,
                                   int64_t D, const void *dq_out,
                                   const void *dk_out, const void *q_out,
                                   const void *k_out, const float *q_rinv,
                                   const float *k_rinv,
                                   const float *cos_table,
                                   const float *sin_table, int64_t n_freq,
                                   int64_t table_ld, void *dq,
                                   const int64_t *dq_strides, void *dk,
                                   const int64_t *dk_strides,
                                   qdl_stream_t stream);

/*
 * Forward with the Q/K prologue folded into the attention kernel's loads:
 *   q' = l2_normalize(apply_unitary_rope(q, c, s)), k' likewise (exactly as
 *   qdl_flash_born_qk_prologue_fwd computes them), then Born attention of
 *   (q', k', v) as qdl_flash_born_fwd computes it.
 * q, k: raw rows with (b, h, t) element strides (q_strides, k_strides: host
 * arrays of 3, unit stride along D), e.g. the (B, T, H, D) projection output;
 * v, out: contiguous (B, H, T, D); the tables and norm_eps as for the
 * prologue; scale, doc_ids, is_causal, window_size, eps as for the forward.
 * Also writes q_out, k_out (contiguous (B, H, T, D), the normalised rows) and
 * q_rinv, k_rinv (1/norm per row), which the backward needs.  For bf16 with
 * D == 64 and no window (with document ids: no window or a causal one), the
 * keys are normalised by the prologue kernel (keys only) and the attention
 * kernel normalises each query block in registers as it loads it, so the
 * normalised queries are never read back from memory; other cases run the
 * prologue kernel on both and then the attention kernels.  The results are those of the two separate calls, bit
 * for bit.  q_rinv and k_rinv may be NULL when no backward follows: then
 * neither 1/norm is written, and q_out is scratch (the one-kernel path does
 * not write it).
 * Replaces the apply_unitary_rope + l2_normalize calls on Q and K
 * (attention.py:583-589) together with the flash_born_attention call that
 * consumes them (attention.py:704-713, flash_born.py:475-513).
 */
int qdl_flash_born_fwd_qk_prologue(int dtype, int64_t B, int64_t H, int64_t T,
                                   int64_t D, const void *q,
                                   const int64_t *q_strides, const void *k,
                                   const int64_t *k_strides, const void *v,
                                   const float *cos_table,
                                   const float *sin_table, int64_t n_freq,
                                   int64_t table_ld, double norm_eps,
                                   const float *scale, int64_t n_scale,
                                   const int32_t *doc_ids, int is_causal,
                                   int64_t window_size, double eps, void *out,
                                   float *z, void *q_out, void *k_out,
                                   float *q_rinv, float *k_rinv,
                                   qdl_stream_t stream);

/*
 * Packed sequences with grouped heads: q, out, dout, dq are (n_q, H, D) rows of
 * tokens, k, v, dk, dv (n_k, h_kv, D), and `sequences` sequences share them:
 * sequence s owns the query rows cu_q[s] .. cu_q[s+1] - 1 and the key rows
 * cu_k[s] .. cu_k[s+1] - 1 (sequences + 1 int32 starts each in device memory,
 * never decreasing, the first 0, values past the rows are cut).  H is a
 * multiple of h_kv; query head h reads key head h / (H / h_kv).  Query i of a
 * sequence of len_q queries and len_k keys stands at position
 * i + len_k - len_q: causality shows it the keys up to its position, a window
 * those less than window_size before it.  Rows that see no key, and rows behind
 * the last sequence, have zero outputs and gradients, and so have rows whose
 * (sum of weights + eps) / scale^2 lies below fp32's normal range, 2^-126.
 *
 * q, k, v, dout have unit stride along D and *_strides (token, head) in
 * elements, multiples of 16 bytes (a token's at least D, under 2^24 bytes);
 * out, dq, dk, dv are contiguous; z is (H, n_q) fp32, NULL in the forward if no
 * backward follows.  scale == NULL takes scale_value.  The weights of fp16 rows are scaled by a power of two of the
 * row's own, so overlaps of any size keep their weight.
 * The backward's dk and dv are summed over the heads of a group in a fixed
 * order; dk == dv == NULL, dscale == NULL: not wanted.  struct_bytes: sizeof
 * the block.
 */
typedef struct qdl_born_packed_call {
    int64_t struct_bytes;
    int64_t dtype, sequences, n_q, n_k, H, h_kv, D;
    const void *q, *k, *v;
    int64_t q_strides[2], k_strides[2], v_strides[2];
    void *out; /* written by the forward, read by the backward */
    float *z;
    const int32_t *cu_q, *cu_k;
    const float *scale;
    int64_t n_scale;
    double scale_value;
    int64_t is_causal, window_size;
    double eps;
    /* backward */
    const void *dout;
    int64_t dout_strides[2];
    void *dq, *dk, *dv;
    float *dscale;
    void *workspace;
    int64_t workspace_bytes;
} qdl_born_packed_call;

int qdl_flash_born_packed_forward_call(const qdl_born_packed_call *call, qdl_stream_t stream);
int64_t qdl_flash_born_packed_workspace_size(const qdl_born_packed_call *call); /* the backward's; 0 for an invalid block */
int qdl_flash_born_packed_backward_call(const qdl_born_packed_call *call, qdl_stream_t stream);

/*
 * A paged cache: k_cache, v_cache hold cache_pages pages of page_size tokens of
 * h_kv heads of D values, *_cache_strides (page, token, head) in elements,
 * multiples of 16 bytes, unit stride along D.  Key j of sequence b is token
 * j % page_size of page block_table[b * table_ld + j / page_size] (int32 in
 * device memory, `pages` columns).  A table entry outside [0, cache_pages) is a
 * missing page: its keys are not seen, nothing is written to it.
 * cache_lens: int32 tokens of each sequence, cut to what its table holds.
 */

/*
 * Attention of one new token per sequence: q (B, H, D) with strides (sequence,
 * head), out (B, H, D) contiguous.  The token is the last of its sequence's
 * cache_lens keys and sees all of them, or the last window_size.  The keys are
 * split over workgroups and joined in order; the workspace's size is the size
 * function's for the same sizes (weighed: key_weight != NULL).
 * key_weight != NULL: (B, h_kv, weight_len) fp32 with weight_strides (sequence,
 * head), to which the sum over the group's heads of p_j / Z is added for every
 * visible key j < weight_len.
 */
typedef struct qdl_born_paged_call {
    int64_t struct_bytes;
    int64_t dtype, B, H, h_kv, D;
    const void *q;
    int64_t q_strides[2];
    void *out;
    const void *k_cache, *v_cache;
    int64_t k_cache_strides[3], v_cache_strides[3];
    int64_t cache_pages, page_size;
    const int32_t *block_table;
    int64_t pages, table_ld;
    const int32_t *cache_lens;
    const float *scale;
    int64_t n_scale;
    double scale_value;
    int64_t window_size;
    double eps;
    float *key_weight;
    int64_t weight_strides[2], weight_len;
    void *workspace;
    int64_t workspace_bytes;
} qdl_born_paged_call;

int64_t qdl_flash_born_paged_workspace_size(int64_t B, int64_t H, int64_t h_kv, int64_t D, int64_t pages,
                                            int64_t page_size, int64_t window_size, int weighed);
int qdl_flash_born_paged_forward_call(const qdl_born_paged_call *call, qdl_stream_t stream);

/*
 * Append: n tokens' queries (n, H, D), keys and values (n, h_kv, D), strides
 * (token, head).  The queries and keys are rotated by row positions[t] of the
 * tables (NULL: the token's slot; rows past the tables take their last) and
 * normalised, x' = y / sqrt(sum y^2 + eps), in fp32 and rounded once; q_out is
 * (n, H, D) contiguous, the keys and the values go to their slots of the cache.
 * cu_seqlens: B + 1 starts of the sequences' new tokens, or NULL: one each
 * (n == B).  cache_lens counts the new tokens, so token t of sequence s goes to
 * slot cache_lens[s] - (cu_seqlens[s+1] - t).  Tokens of no sequence have zero
 * queries; slots without a page are not written.  cos_table NULL: no rotation;
 * tables and n_freq as for the Q/K prologue, table_rows rows.  D: a multiple of 8.
 */
typedef struct qdl_born_append_call {
    int64_t struct_bytes;
    int64_t dtype, n, B, H, h_kv, D;
    const void *q, *k, *v;
    int64_t q_strides[2], k_strides[2], v_strides[2];
    void *q_out;
    void *k_cache, *v_cache;
    int64_t k_cache_strides[3], v_cache_strides[3];
    int64_t cache_pages, page_size;
    const int32_t *block_table;
    int64_t pages, table_ld;
    const int32_t *cache_lens, *cu_seqlens;
    const float *cos_table, *sin_table;
    int64_t table_rows, n_freq, freq_ld;
    const int32_t *positions;
    double eps;
} qdl_born_append_call;

int qdl_flash_born_cache_append_call(const qdl_born_append_call *call, qdl_stream_t stream);

/*
 * Evict: every sequence longer than `budget` keeps, for each key head, its last
 * min(recent, budget) keys and of the others those with the greatest
 * key_weight, budget in all, ties to the lowest index (NaN above all numbers;
 * keys at weight_len and after have weight 0).  They keep their order.
 * kept (B, h_kv, budget): the kept keys' old slots, -1 behind the last;
 * weight_out (B, h_kv, weight_len): their weights, 0 behind the last;
 * lens_out (B): min(cache_lens, budget).  None of the three may overlap an
 * input.
 * The kept rows of K and V move to slots 0, 1, ... of out_table's pages
 * (out_pages columns), none of which may be a page of block_table, or, with
 * out_table NULL, of block_table's own.  Rows behind the last kept one stay as
 * they were; a row kept from a missing page arrives as zeros.
 */
typedef struct qdl_born_evict_call {
    int64_t struct_bytes;
    int64_t dtype, B, h_kv, D;
    void *k_cache, *v_cache;
    int64_t k_cache_strides[3], v_cache_strides[3];
    int64_t cache_pages, page_size;
    const int32_t *block_table;
    int64_t pages, table_ld;
    const int32_t *cache_lens;
    const float *key_weight;
    int64_t weight_strides[2], weight_len;
    int64_t budget, recent;
    const int32_t *out_table;
    int64_t out_pages, out_table_ld;
    float *weight_out;
    int32_t *lens_out, *kept;
} qdl_born_evict_call;

int qdl_flash_born_cache_evict_call(const qdl_born_evict_call *call, qdl_stream_t stream);

/*
 * A paged cache in 4 bits.  A row (one head of one token) holds W = 32 nb
 * columns, D rounded up to whole blocks of 32: 16 nb bytes of codes (the lower
 * nibble is the even column; sign, two exponent bits, one mantissa bit: 0, .5,
 * 1, 1.5, 2, 3, 4, 6) and nb scale bytes e; a value is its code times 2^(e - 127),
 * e = 255: not a number.  k, v: cache_pages pages of page_size tokens of h_kv
 * heads; *_strides (page, token, head) in bytes, under 2^32, the codes' multiples
 * of 16, and unit strides within a row.  Pages, tables and lengths as above.
 */
typedef struct qdl_born_fp4_cache {
    void *k, *v, *k_scale, *v_scale;
    int64_t k_strides[3], v_strides[3], k_scale_strides[3], v_scale_strides[3];
    int64_t cache_pages, page_size;
    const int32_t *block_table;
    int64_t pages, table_ld;
    const int32_t *cache_lens;
} qdl_born_fp4_cache;

/*
 * Append, as qdl_flash_born_cache_append_call, the keys and values stored in 4
 * bits: e is the least with max |x| <= 7 2^(e - 127) over the block, at least 1,
 * the codes are nearest, halfway to even, at most 6; blocks with an infinity, a
 * NaN or a magnitude past 7 2^125 get e = 255.  Keys are rotated and normalised
 * in 64 bits, queries in fp32.
 */
typedef struct qdl_born_fp4_append_call {
    int64_t struct_bytes;
    int64_t dtype, n, B, H, h_kv, D;
    const void *q, *k, *v;
    int64_t q_strides[2], k_strides[2], v_strides[2];
    void *q_out;
    qdl_born_fp4_cache cache;
    const int32_t *cu_seqlens;
    const float *cos_table, *sin_table;
    int64_t table_rows, n_freq, freq_ld;
    const int32_t *positions;
    double eps;
} qdl_born_fp4_append_call;

int qdl_flash_born_fp4_append_call(const qdl_born_fp4_append_call *call, qdl_stream_t stream);

/*
 * Read: the values of n rows of a packed batch, k_out and v_out (n, h_kv, D)
 * contiguous.  Rows cu_seqlens[s] .. cu_seqlens[s+1] - 1 are the last keys of
 * sequence s; rows of no sequence, and of missing pages, are zeros.
 */
typedef struct qdl_born_fp4_read_call {
    int64_t struct_bytes;
    int64_t dtype, n, B, h_kv, D;
    void *k_out, *v_out;
    qdl_born_fp4_cache cache;
    const int32_t *cu_seqlens;
} qdl_born_fp4_read_call;

int qdl_flash_born_fp4_read_call(const qdl_born_fp4_read_call *call, qdl_stream_t stream);

/*
 * Attention over the cache: q (n, H, D) with strides (token, head), out (n, H,
 * D) contiguous, both of dtype.  cu_seqlens: B + 1 starts of the sequences'
 * tokens, or NULL: one each (n == B).  A sequence's tokens stand at the last of
 * its keys: its i-th of m is at position cache_lens - m + i and sees the keys up
 * to there, or the last window_size of them.  Tokens that see no key, and those
 * of no sequence, get zeros; a key with a block of e = 255 makes NaN of every
 * row that sees it.  B up to 65536.  The workspace's size is the size function's for the same
 * sizes (packed: cu_seqlens != NULL; weighed: 0 without key_weight, else its
 * weight_len, where 1 stands for any: H fp32 values for each of the weight_len
 * keys a sequence, or of as many as the table has room for); it is 0 for sizes
 * that the call refuses.
 * key_weight, only where cu_seqlens is NULL: as for qdl_flash_born_paged_forward_call.
 */
typedef struct qdl_born_fp4_paged_call {
    int64_t struct_bytes;
    int64_t dtype, n, B, H, h_kv, D;
    const void *q;
    int64_t q_strides[2];
    void *out;
    qdl_born_fp4_cache cache;
    const int32_t *cu_seqlens;
    const float *scale;
    int64_t n_scale;
    double scale_value;
    int64_t window_size;
    double eps;
    float *key_weight;
    int64_t weight_strides[2], weight_len;
    void *workspace;
    int64_t workspace_bytes;
} qdl_born_fp4_paged_call;

int64_t qdl_flash_born_fp4_paged_workspace_size(int64_t n, int64_t B, int64_t H, int64_t h_kv, int64_t D, int64_t pages,
                                                int64_t page_size, int64_t window_size, int packed, int weighed);
int qdl_flash_born_fp4_paged_forward_call(const qdl_born_fp4_paged_call *call, qdl_stream_t stream);

/* Evict, as qdl_flash_born_cache_evict_call.  A row kept from a missing page arrives as zeros. */
typedef struct qdl_born_fp4_evict_call {
    int64_t struct_bytes;
    int64_t B, h_kv, D;
    qdl_born_fp4_cache cache;
    const float *key_weight;
    int64_t weight_strides[2], weight_len;
    int64_t budget, recent;
    const int32_t *out_table;
    int64_t out_pages, out_table_ld;
    float *weight_out;
    int32_t *lens_out, *kept;
} qdl_born_fp4_evict_call;

int qdl_flash_born_fp4_evict_call(const qdl_born_fp4_evict_call *call, qdl_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* QDL_FLASH_BORN_H */
