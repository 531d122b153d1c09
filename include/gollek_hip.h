/*
 * gollek_hip.h -- C ABI of the MI355X (gfx950) GGUF quantized linear-layer
 * library, libgollek_hip.so.
 *
 * The library is the native side of a drop-in for gollek's Java GGUF tensor
 * runtime (RT/ = runner/gguf/gollek-gguf-core/src/main/java/tech/kayys/gollek/
 * gguf/runtime/).  The Java facade RT/GgufTensorOps keeps its signatures; an
 * FFM (java.lang.foreign) binding calls these functions from inside
 * RT/GgufMatVec.rows (RT/GgufMatVec.java:55-96) for ggml type ids 2 (Q4_0),
 * 8 (Q8_0), 12 (Q4_K), 13 (Q5_K) and 14 (Q6_K), ahead of the prepared and raw
 * Java routes.
 *
 * Conventions (those of the reference's own native bridge,
 * runner/gguf/gguf-fast-bridge/gollek_gguf_fast.cpp:672-800):
 *   - plain C types only: pointers, int32/int64 sizes, floats;
 *   - functions returning int return GOLLEK_HIP_OK (0) or a negative code;
 *     handle constructors return NULL on failure;
 *   - a message is written to the caller's `err` buffer (NUL-terminated,
 *     truncated to err_len) when err != NULL and err_len > 0;
 *   - the Java adapter maps codes back to the reference's exceptions:
 *     NULL -> NullPointerException (RT/GgufMatVec.java:32-35),
 *     ARG -> IllegalArgumentException (RT/GgufMatVec.java:65-71, :196-200;
 *            RT/GgufTensorOps.java:652-656; GC/core/GgmlType.java:70-81),
 *     UNSUPPORTED -> UnsupportedOperationException (RT/GgufRowDot.java:77-82,
 *            RT/GgufRowDequantizer.java:275),
 *     DEVICE / NOMEM -> IllegalStateException (no reference counterpart: the
 *            Java path has no device).
 *
 * Threading: every function may be called from any thread.  A weight handle
 * serialises its host-buffer calls with its own mutex (as the reference
 * bridge does per handle, gollek_gguf_fast.cpp:42) and runs them on its own
 * HIP stream; they return only when the output is in host memory.  The
 * *_device functions are asynchronous on the caller's stream and take device
 * pointers.
 */
#ifndef GOLLEK_HIP_H
#define GOLLEK_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GOLLEK_HIP_OK 0
#define GOLLEK_HIP_ERR_NULL (-1)
#define GOLLEK_HIP_ERR_ARG (-2)
#define GOLLEK_HIP_ERR_UNSUPPORTED (-3)
#define GOLLEK_HIP_ERR_DEVICE (-4)
#define GOLLEK_HIP_ERR_NOMEM (-5)

/* ggml type ids accepted by this library (GC/core/GgmlType.java:11,16,21).  The
 * *_device mat-vec of Q5_K / Q6_K needs x 16-byte aligned and Q5_K weights
 * 4-byte aligned (else DEVICE). */
#define GOLLEK_HIP_Q4_0 2
#define GOLLEK_HIP_Q8_0 8
#define GOLLEK_HIP_Q4_K 12
#define GOLLEK_HIP_Q5_K 13 /* GC/core/GgmlType.java:22 */
#define GOLLEK_HIP_Q6_K 14 /* GC/core/GgmlType.java:23 */

/* Opaque device-resident weight matrix. */
typedef struct gollek_hip_weight gollek_hip_weight;

/* ABI version (major * 10000 + minor * 100 + patch).  No reference
 * counterpart; lets the Java binding refuse a mismatched library. */
int32_t gollek_hip_version(void);

/* Select and initialise a GPU.  Replaces the reference bridge's one-time
 * backend set-up in gollek_gguf_open (gollek_gguf_fast.cpp:692-700).
 * Calling it again with the same device is a no-op. */
int32_t gollek_hip_init(int32_t device, char *err, size_t err_len);

/* Thread-local copy of the last error message of this thread ("" if none). */
const char *gollek_hip_last_error(void);

/* Thread-local status code of this thread's last call (GOLLEK_HIP_OK after a
 * success).  Lets a caller map a NULL handle back to the exception type. */
int32_t gollek_hip_last_status(void);

/* Copy a GGUF row-major matrix (rows x cols, cols contiguous; row_bytes =
 * cols / block_size * block_bytes) from host memory to a device handle.  The
 * bytes are the tensor's bytes at dataStart + offset in the mmapped file
 * (RT/GgufTensorData.java:40, GC/loader/GGUFReader.java:30-37).  Replaces the
 * reference's prepared-matrix build at model load (RT/GgufPreparedMatrixStore
 * .java:120-127 via PRG/JavaNativeGgufBackend.java:157-180): the layout stays
 * the packed GGUF layout, only its residency changes.  NULL on failure. */
gollek_hip_weight *gollek_hip_weight_upload(int32_t type_id, const void *host_bytes,
                                            int64_t rows, int64_t cols, int64_t row_bytes,
                                            char *err, size_t err_len);

/* Wrap GGUF bytes that are already in device memory (borrowed: the caller
 * keeps ownership and must outlive the handle).  Same validation as upload. */
gollek_hip_weight *gollek_hip_weight_wrap_device(int32_t type_id, const void *device_bytes,
                                                 int64_t rows, int64_t cols,
                                                 int64_t row_bytes, char *err,
                                                 size_t err_len);

/* Build the handle's prepared mat-vec layout: a second device copy of the
 * matrix in which every workgroup's block of rows is stored superblock
 * column by column, the order the matrix-core column kernels read (Q4_K,
 * Q8_0, Q4_0 and Q5_K with K up to 16384 and at most 64 / 32 / 64 / 48 rows
 * per CU; measured 7.8 us against 8.8 us for Q4_K 14336 x 4096).  Later full mat-vecs
 * (row_count == rows) on the handle read it; every other entry point keeps
 * reading the GGUF bytes.  The layout follows the device's CU count at the
 * time of the call; a no-op (OK) for other shapes.  The copy is a snapshot:
 * a caller that rewrites a borrowed buffer (gollek_hip_weight_wrap_device)
 * after this call must call gollek_hip_weight_unprepare, or this again,
 * before the next full mat-vec.  The copy costs the matrix's bytes a second
 * time in device memory.
 * Call it before the handle's device mat-vecs start, or with none in
 * flight: a call that finds a copy for another partition frees it, and the
 * _device entry points read the copy on the caller's stream without the
 * handle's lock.
 * Replaces the reference's prepared-matrix build at model load
 * (RT/GgufPreparedMatrixStore.java:120-127 via PRG/JavaNativeGgufBackend
 * .java:157-180), which likewise keeps a prepared copy beside the raw
 * bytes.  Freed with the handle.  Device memory exhausted -> NOMEM. */
int32_t gollek_hip_weight_prepare(gollek_hip_weight *weight, char *err, size_t err_len);

/* Free the prepared copy of gollek_hip_weight_prepare, if any (OK when there
 * is none); later full mat-vecs read the GGUF bytes again, with identical
 * results.  Gives a caller the device memory back while keeping the handle,
 * as the reference's per-family prepared-cache clear keeps the raw tensor
 * (RT/GgufPreparedMatrixStore.java:129-131).  Same rule as prepare: no
 * _device call on the handle may be in flight. */
int32_t gollek_hip_weight_unprepare(gollek_hip_weight *weight, char *err, size_t err_len);

/* Keep only the prepared layout: free the handle's GGUF copy, so the packed
 * bytes are held once.  Full and prefix mat-vecs (matvec_rows, dot_row and
 * the _device form) then run the full mat-vec from the layout, so a prefix
 * or a single row returns exactly the full call's bits for its rows;
 * dequantize_rows gathers the rows' bytes back from the layout first (the
 * same bytes, so the same bits).  The GEMM entry points run up to four
 * rows of X (8-byte aligned) on the layout when K <= 4096, two up to K =
 * 16384; other GEMM shapes
 * and the MoE entry points read GGUF rows and return UNSUPPORTED for a
 * compacted handle;
 * gollek_hip_weight_unprepare rebuilds the GGUF copy (and frees the
 * layout).  Needs a prepared handle that owns its bytes: a borrowed
 * (wrap_device) buffer -> ARG, no layout -> UNSUPPORTED.  Replaces keeping
 * the raw tensor beside the prepared one (RT/GgufPreparedMatrixStore.java:
 * 120-131 keeps one prepared representation per tensor).  No _device call
 * on the handle may be in flight; the _device entries of a compacted handle
 * share temporaries of the handle (grown on demand), so they must not
 * overlap on one handle. */
int32_t gollek_hip_weight_compact(gollek_hip_weight *weight, char *err, size_t err_len);

/* Release a handle (device memory it owns, its stream and staging buffers).
 * Replaces clearPreparedMatrixCaches on backend close
 * (PRG/JavaNativeGgufBackend.java:139-143).  NULL is ignored. */
void gollek_hip_weight_free(gollek_hip_weight *weight);

/* Shape of a handle; any out pointer may be NULL. */
int32_t gollek_hip_weight_info(const gollek_hip_weight *weight, int32_t *type_id,
                               int64_t *rows, int64_t *cols, int64_t *row_bytes);

/* ---- host-buffer entry points (synchronous; the Java drop-in) ---------- */

/* Dequantize rows [row0, row0 + nrows) into dst (nrows * cols floats,
 * dst_len >= that), bit-exact with RT/GgufRowDequantizer.dequantizeRow.
 * Replaces GgufTensorOps.dequantizeRow (RT/GgufTensorOps.java:636-642) when
 * nrows == 1; row outside [0, rows) -> ARG (:652-656). */
int32_t gollek_hip_dequantize_rows(gollek_hip_weight *weight, int64_t row0, int64_t nrows,
                                   float *dst, int64_t dst_len, char *err, size_t err_len);

/* out[0] = dot(row, x).  Replaces GgufTensorOps.dotRow
 * (RT/GgufTensorOps.java:644-650): x_len >= cols (extra entries ignored),
 * row outside [0, rows) -> ARG. */
int32_t gollek_hip_dot_row(gollek_hip_weight *weight, int64_t row, const float *x,
                           int64_t x_len, float *out, char *err, size_t err_len);

/* y[r] = sum_k W[r, k] x[k] for r < row_count (a prefix of the rows).
 * Replaces GgufTensorOps.matVecRows (RT/GgufTensorOps.java:666-674) and,
 * with row_count = rows, matVec / matVecParallel (:658-664), with the
 * checks of RT/GgufMatVec.java:63-75, :196-200: row_count outside
 * [0, rows] -> ARG, y_len < row_count -> ARG, x_len < cols -> ARG,
 * row_count == 0 -> no-op. */
int32_t gollek_hip_matvec_rows(gollek_hip_weight *weight, const float *x, int64_t x_len,
                               float *y, int64_t y_len, int64_t row_count, char *err,
                               size_t err_len);

/* Y[m, n] = sum_k X[m, k] W[n, k] (Y = X W^T, the Linear convention of
 * runner/safetensor/gollek-safetensor-core/src/main/java/tech/kayys/gollek/
 * safetensor/core/tensor/AccelOps.java:370-376) for a weight of any type
 * this library takes (on bf16 matrix cores; Q6_K rows of an odd superblock
 * count on fp32 ones over their exactly dequantized values), X given as
 * m x cols bf16 bit patterns (row-major), Y m x rows fp32.  Small-M prefill
 * and batched decode.  The reference has no GGUF GEMM: it runs m independent
 * RT/GgufTensorOps.matVecRows calls (RT/GgufTensorOps.java:666-674), which
 * this replaces.  x_len < m * cols or y_len < m * rows -> ARG. */
int32_t gollek_hip_gemm_bf16(gollek_hip_weight *weight, const uint16_t *x_bf16, int64_t x_len,
                             int64_t m, float *y, int64_t y_len, char *err, size_t err_len);

/* ---- the linear layer ---------------------------------------------------- */

/* Element types of a linear layer's output and of logits (ggml type ids). */
#define GOLLEK_HIP_F32 0
#define GOLLEK_HIP_F16 1
#define GOLLEK_HIP_BF16 30

/* Activations: relu max(v, 0); silu v / (1 + exp(-v)); gelu v Phi(v) (by erf);
 * gelu_tanh its tanh form 0.5 v (1 + tanh(sqrt(2 / pi) (v + 0.044715 v^3))). */
#define GOLLEK_HIP_ACT_NONE 0
#define GOLLEK_HIP_ACT_RELU 1
#define GOLLEK_HIP_ACT_SILU 2
#define GOLLEK_HIP_ACT_GELU 3
#define GOLLEK_HIP_ACT_GELU_TANH 4

/* The GEMM with what a model does with its result:
 *   Y[m, n] = act(sum_k X[m, k] W[n, k] + bias[n]) * mul[m, n] + residual[m, n]
 * in fp32, rounded once to y_type (F32, F16 or BF16; nearest, ties to even).
 * bias (`rows` floats), mul and residual (m x rows of y_type) may each be NULL
 * and are then left out.  The sums are gollek_hip_gemm_bf16's for the same
 * weight, X and m (bit for bit where neither splits K); one row of X, 16-byte
 * aligned, has gollek_hip_matvec_rows's of that row widened to fp32 with a Q6_K
 * weight of a multiple of 2048 columns up to 14336 (unless it splits K) and with
 * a Q4_K one of up to 4096 columns and too many rows for the mat-vec's column
 * layout.
 * A gated FFN is two calls: the up product, then the gate's with
 * activation SILU and mul = the up product's Y.  The reference adds biases and
 * residuals in Java after its linear (AccelOps.java:370-376).
 * The host form takes packed matrices; x_len < m * cols or y_len < m * rows ->
 * ARG (mul and residual hold y_len elements too).  An unknown activation -> ARG,
 * another y_type -> UNSUPPORTED; the checks of gollek_hip_gemm_bf16 apply.
 * m == 0 is a no-op. */
int32_t gollek_hip_linear(gollek_hip_weight *weight, const uint16_t *x_bf16, int64_t x_len, int64_t m,
                          const float *bias, int32_t activation, const void *mul, const void *residual, void *y,
                          int32_t y_type, int64_t y_len, char *err, size_t err_len);

/* Device workspace bytes with which gollek_hip_linear_device splits K as far as
 * it pays (0: a call of m rows never splits): for Q8_0 and Q4_0 up to some
 * hundred MB for long prompts, for the others partials of at most 16 MiB beyond
 * the first; -1 for a NULL weight or m out of range. */
int64_t gollek_hip_linear_workspace_bytes(const gollek_hip_weight *weight, int64_t m);

/* Device variant, asynchronous on `stream`, which belongs to the weight's
 * device; allocates nothing, so it can be captured into a graph.  The strides
 * are elements between rows, at least `rows` (0: packed).  Y may be mul or
 * residual (the same address and stride), or another column range of one wider
 * matrix; any other overlap of Y with mul or residual, and any of Y with X, bias
 * or workspace, -> ARG (the gaps between Y's rows counted in; Y must not overlap
 * the weight either).  Elements of Y's rows past column `rows` are left as they
 * are.  Pointers are aligned to their elements (else
 * ARG).  workspace (256-byte aligned, else ARG) may be smaller than
 * gollek_hip_linear_workspace_bytes, or NULL: the call splits less, which
 * changes Y by the rounding of the sums' order alone.  A larger one changes
 * nothing: bytes past those are not touched, so one workspace may serve calls of
 * different needs.  The bytes that the call may use must not overlap X, bias, mul
 * or residual (-> ARG).  Calls that share a workspace must not overlap. */
int32_t gollek_hip_linear_device(gollek_hip_weight *weight, const uint16_t *x_bf16, int64_t m, const float *bias,
                                 int32_t activation, const void *mul, int64_t mul_stride, const void *residual,
                                 int64_t residual_stride, void *y, int32_t y_type, int64_t y_stride, void *workspace,
                                 int64_t workspace_bytes, void *stream, char *err, size_t err_len);

/* Grouped MoE expert FFN over expert weights of any type this library takes
 * (Q4_0, Q8_0, Q4_K, Q5_K, Q6_K; gate, up and down may differ, as in Q4_K_M
 * files whose ffn_down_exps are Q6_K in some layers), stacked as GGUF stores
 * them:
 * gate and up have n_experts * inter rows of `hidden` columns, down has
 * n_experts * hidden rows of `inter` columns.  For each token t (x row-major
 * tokens x hidden) and route j < top_k (ids / weights row-major tokens x
 * top_k): out[t] += weights[t,j] * down_e(silu(gate_e x_t) * up_e x_t) with
 * e = ids[t,j], accumulated in route order; a route whose id is outside
 * [0, n_experts) or whose weight is 0 is skipped.  Replaces the per-(token,
 * route) expert loop of runner/safetensor/gollek-safetensor-engine/src/main/
 * java/tech/kayys/gollek/safetensor/engine/generation/moe/MoeForwardPass.java:
 * 217-240 with :461-472 (swigluFfn: .../engine/forward/
 * DirectForwardFfnService.java:40-61), reading each used expert once.
 * Other weight types -> UNSUPPORTED; gate rows not a multiple of n_experts,
 * shapes that disagree, or tokens * top_k above 2^24 -> ARG. */
int32_t gollek_hip_moe_grouped(gollek_hip_weight *gate, gollek_hip_weight *up,
                               gollek_hip_weight *down, int64_t n_experts, const float *x,
                               int64_t tokens, const int32_t *ids, const float *weights,
                               int64_t top_k, float *out, int64_t out_len, char *err,
                               size_t err_len);

/* Device workspace bytes gollek_hip_moe_grouped_device needs. */
int64_t gollek_hip_moe_workspace_bytes(int64_t tokens, int64_t top_k, int64_t hidden,
                                       int64_t inter, int64_t n_experts);

/* ---- device-buffer entry points (asynchronous on `stream`) ------------- */
/* `stream` is a hipStream_t passed as void* (NULL = the null stream).  All
 * pointers are device pointers.  Same semantics as the host versions. */

int32_t gollek_hip_dequantize_rows_device(gollek_hip_weight *weight, int64_t row0,
                                          int64_t nrows, float *dst, void *stream, char *err,
                                          size_t err_len);

int32_t gollek_hip_matvec_device(gollek_hip_weight *weight, const float *x, float *y,
                                 int64_t row_count, void *stream, char *err, size_t err_len);

/* Shapes whose output tiles leave CUs idle (few 128 x 128 tiles for the
 * chip) are split over K into partial tiles held in a workspace of the
 * handle, allocated at the first such call (below 16 MiB on 256 CUs) and
 * freed with the handle; splitting calls on one handle share it and must not
 * overlap (calls on different handles may).  A y that is not 16-byte aligned
 * runs unsplit. */
int32_t gollek_hip_gemm_bf16_device(gollek_hip_weight *weight, const uint16_t *x_bf16, int64_t m,
                                    float *y, void *stream, char *err, size_t err_len);

/* gollek_hip_gemm_bf16_device without any allocation.  No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops).  The split-K partial tiles
 * go to a static per-GPU scratch of 16 MiB (held from library load until the
 * process ends; enough for every shape on a 256-CU MI355X) instead of the
 * handle's lazily allocated workspace; a shape whose splits would need more
 * is split less, down to none.  All calls on one GPU share that scratch, so
 * calls that overlap on a GPU race.  Same checks and results as
 * gollek_hip_gemm_bf16_device. */
int32_t gollek_hip_gemm_bf16_device_noalloc(gollek_hip_weight *weight, const uint16_t *x_bf16,
                                            int64_t m, float *y, void *stream, char *err,
                                            size_t err_len);

/* `workspace` (device, workspace_bytes >= gollek_hip_moe_workspace_bytes) is
 * scratch owned by the caller; calls sharing one workspace must not overlap. */
int32_t gollek_hip_moe_grouped_device(gollek_hip_weight *gate, gollek_hip_weight *up,
                                      gollek_hip_weight *down, int64_t n_experts, const float *x,
                                      const int32_t *ids, const float *weights, int64_t tokens,
                                      int64_t top_k, float *out, void *workspace,
                                      int64_t workspace_bytes, void *stream, char *err,
                                      size_t err_len);

/* ---- MoE router and the routed block ------------------------------------ */
/* SFE/ = runner/safetensor/gollek-safetensor-engine/src/main/java/tech/kayys/
 * gollek/safetensor/engine/. */

/* Router scoring (SFE/generation/moe/MoeForwardPass.java:174-197): the
 * reference picks sigmoid when the model type contains "qwen" or "moe",
 * softmax otherwise; the caller passes that choice. */
#define GOLLEK_HIP_ROUTER_SOFTMAX 0
#define GOLLEK_HIP_ROUTER_SIGMOID 1

/* Per token t (logits row-major tokens x n_experts, the router linear's
 * output): probabilities by `scoring` (sigmoid 1 / (1 + exp(-l)); softmax
 * exp(l - max) / sum with exp in double and float sums in expert order),
 * then the top_k experts in descending probability order, ties in index
 * order, and their probabilities divided by their float sum when that sum
 * is > 0 -> ids / weights (row-major tokens x top_k).  Ranks past n_experts
 * get id 0, weight 0.  Replaces MoeForwardPass.java:174-203 with selectTopK
 * (:286-306), bit for bit.  n_experts or top_k outside [1, 4096], an unknown
 * scoring -> ARG.  Synchronous; allocates device memory per call (the
 * _device variant does not). */
int32_t gollek_hip_moe_select_topk(const float *logits, int64_t tokens, int64_t n_experts,
                                   int64_t top_k, int32_t scoring, int32_t *ids, float *weights,
                                   char *err, size_t err_len);
int32_t gollek_hip_moe_select_topk_device(const float *logits, int64_t tokens, int64_t n_experts,
                                          int64_t top_k, int32_t scoring, int32_t *ids,
                                          float *weights, void *stream, char *err,
                                          size_t err_len);

/* The routed MoE block: gollek_hip_moe_select_topk on `logits` followed by
 * gollek_hip_moe_grouped with the ids and weights it chose, on one stream
 * (MoeForwardPass.java:174-240 after the router linear).  The shared expert
 * (:240-247) follows with gollek_hip_moe_shared_expert on the same `out`.
 * Checks of both calls apply. */
int32_t gollek_hip_moe_block(gollek_hip_weight *gate, gollek_hip_weight *up,
                             gollek_hip_weight *down, int64_t n_experts, const float *x,
                             int64_t tokens, const float *logits, int64_t top_k, int32_t scoring,
                             float *out, int64_t out_len, char *err, size_t err_len);
/* Device variant: also writes the chosen ids / weights (device, tokens x
 * top_k) and takes the grouped FFN's workspace from the caller
 * (gollek_hip_moe_workspace_bytes; calls sharing it must not overlap). */
int32_t gollek_hip_moe_block_device(gollek_hip_weight *gate, gollek_hip_weight *up,
                                    gollek_hip_weight *down, int64_t n_experts, const float *x,
                                    const float *logits, int64_t tokens, int64_t top_k,
                                    int32_t scoring, int32_t *ids, float *weights, float *out,
                                    void *workspace, int64_t workspace_bytes, void *stream,
                                    char *err, size_t err_len);

/* Routing with what gollek_hip_moe_select_topk has not: logits of type F32, F16
 * or BF16, a bias for balance, groups, and weights as they are.  Per token:
 *   p = softmax(l) or 1 / (1 + exp(-l)) by `scoring`;  c = p + bias (n_experts
 *   floats, NULL: none);
 *   the n_experts / n_groups neighbours of a group make it worth the sum of
 *   their group_top (1 or 2) largest c; the top_groups groups worth most stay;
 *   of their experts the top_k with the largest c, in that order -> ids; ties
 *   (of groups too) go to the lower index, NaN comes first;
 *   weights = p of each (without the bias), divided by their sum if renormalize
 *   and the sum is > 0, times scale.
 * Computed in double and rounded once; ids and weights row-major tokens x
 * top_k.  n_experts in [1, 4096]; n_groups in [1, 64] dividing it, top_groups in
 * [1, n_groups]; top_k in [1, top_groups * n_experts / n_groups]; tokens * top_k up
 * to 2^24 and tokens * n_experts up to 2^30; a finite scale; aligned pointers:
 * else ARG; another logits_type -> UNSUPPORTED.  In the device forms ids and
 * weights must not overlap the logits, the bias or each other (-> ARG).  No reference
 * counterpart: MoeForwardPass.java:174-203 routes by plain scores alone. */
int32_t gollek_hip_moe_route(const void *logits, int32_t logits_type, int64_t tokens, int64_t n_experts,
                             const float *bias, int32_t scoring, int64_t n_groups, int64_t top_groups,
                             int32_t group_top, int64_t top_k, int32_t renormalize, float scale, int32_t *ids,
                             float *weights, char *err, size_t err_len);
int32_t gollek_hip_moe_route_device(const void *logits, int32_t logits_type, int64_t tokens, int64_t n_experts,
                                    const float *bias, int32_t scoring, int64_t n_groups, int64_t top_groups,
                                    int32_t group_top, int64_t top_k, int32_t renormalize, float scale, int32_t *ids,
                                    float *weights, void *stream, char *err, size_t err_len);

/* The MoE block behind that routing: gollek_hip_moe_route_device, then
 * gollek_hip_moe_grouped_device with the ids and weights it chose, on one
 * stream (as gollek_hip_moe_block_device; the checks of both calls apply). */
int32_t gollek_hip_moe_block_routed_device(gollek_hip_weight *gate, gollek_hip_weight *up, gollek_hip_weight *down,
                                           int64_t n_experts, const float *x, const void *logits, int32_t logits_type,
                                           int64_t tokens, const float *bias, int32_t scoring, int64_t n_groups,
                                           int64_t top_groups, int32_t group_top, int64_t top_k, int32_t renormalize,
                                           float scale, int32_t *ids, float *weights, float *out, void *workspace,
                                           int64_t workspace_bytes, void *stream, char *err, size_t err_len);

/* The shared expert, added to the routed output of the same tokens
 * (SFE/generation/moe/MoeForwardPass.java:240-247 with runSharedExpert
 * :418-426 and resolveSharedExpertGate :428-442): for each token t
 *   out[t] = out[t] + g_t * y_t   (the product rounded, then the sum),
 *   y_t = down(silu(gate x_t) * (up x_t)),
 *   g_t = 1 / (1 + (float)exp(-s_t)) with exp in double, s_t = x_t . gate_inp
 *         rounded to float (gate_inp: `hidden` floats, the shared_expert_gate
 *         row); g_t = 1 when gate_inp is NULL (the reference's missing gate).
 * gate / up: inter x hidden, down: hidden x inter, of any types
 * gollek_hip_moe_grouped takes.  Errors as gollek_hip_moe_grouped with one
 * expert (x and out NULL -> NULL; out_len < tokens * hidden -> ARG). */
int32_t gollek_hip_moe_shared_expert(gollek_hip_weight *gate, gollek_hip_weight *up,
                                     gollek_hip_weight *down, const float *gate_inp, const float *x,
                                     int64_t tokens, float *out, int64_t out_len, char *err,
                                     size_t err_len);
/* Device workspace bytes gollek_hip_moe_shared_expert_device needs. */
int64_t gollek_hip_moe_shared_workspace_bytes(int64_t tokens, int64_t hidden, int64_t inter);
/* Device variant (x, gate_inp, out on the device; `workspace` as for
 * gollek_hip_moe_grouped_device, >= gollek_hip_moe_shared_workspace_bytes). */
int32_t gollek_hip_moe_shared_expert_device(gollek_hip_weight *gate, gollek_hip_weight *up,
                                            gollek_hip_weight *down, const float *gate_inp, const float *x,
                                            int64_t tokens, float *out, void *workspace,
                                            int64_t workspace_bytes, void *stream, char *err,
                                            size_t err_len);

/* ---- sampling -------------------------------------------------------------- */

/* One token per row of logits (rows x vocab of type F32, F16 or BF16, rows
 * `logits_stride` elements apart, 0: packed), as the lm_head's product leaves
 * them, with settings per row.  Tokens are ordered by logit, equal ones by
 * index; -inf and NaN logits are no tokens (a grammar's mask).  Per row:
 *   w_i = exp((l_i - max l) / temperature);  temperature <= 0 or NaN keeps the
 *   first token alone;
 *   top_k > 0 keeps the first top_k tokens;  top_p < 1 keeps of these the
 *   shortest prefix whose w add up to at least top_p of theirs (one token at
 *   least);  min_p > 0 keeps of these the ones with w_i >= min(min_p, 1);
 *   the token is the first, in the order of the vocabulary, at which the kept w
 *   add up to more than u times all kept w (u the caller's random number in
 *   [0, 1); below 0 or NaN it counts as 0, from 1 as the last fp32 below it).
 * -> tokens[row] (-1 where a row has no token), probs[row] = its share of the
 * kept w (0 without a token), kept[row] = how many were kept.  temperature (1),
 * top_k, top_p and min_p (off), probs and kept may be NULL.  An infinite logit
 * leaves only the infinite ones with weight.  Weights are summed exactly as
 * multiples of 2^-S, vocab 2^S < 2^62, so a row's token does not depend on
 * the batch around it.
 * rows in [0, 65535], vocab in [1, 4194304], a stride of at least vocab, aligned
 * pointers: else ARG; another logits_type -> UNSUPPORTED.  The host form takes
 * packed logits and copies them up.  No counterpart on the reference's GGUF path
 * (its sampling runs on the logits in host memory). */
int32_t gollek_hip_sample(const void *logits, int32_t logits_type, int64_t rows, int64_t vocab,
                          const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                          const float *u, int32_t *tokens, float *probs, int32_t *kept, char *err, size_t err_len);
/* Device workspace bytes gollek_hip_sample_device needs (-1: out of range).  They
 * never fall as rows or vocab rise: the workspace of the largest batch and
 * vocabulary serves every smaller call. */
int64_t gollek_hip_sample_workspace_bytes(int64_t rows, int64_t vocab);
/* Device variant (every pointer on the device; `workspace` 256-byte aligned and
 * of at least gollek_hip_sample_workspace_bytes, else ARG; calls sharing it must
 * not overlap).  The results and the workspace's bytes must not overlap the
 * logits' rows, a setting or each other (-> ARG), but a result may be a setting's
 * own array.  Allocates nothing: it can be captured into a graph. */
int32_t gollek_hip_sample_device(const void *logits, int32_t logits_type, int64_t rows, int64_t vocab,
                                 int64_t logits_stride, const float *temperature, const int32_t *top_k,
                                 const float *top_p, const float *min_p, const float *u, int32_t *tokens, float *probs,
                                 int32_t *kept, void *workspace, int64_t workspace_bytes, void *stream, char *err,
                                 size_t err_len);

/* The next token of one sequence: the lm_head's mat-vec (gollek_hip_matvec_rows
 * of all rows) and gollek_hip_sample on its result, which stays on the device
 * (a 128k vocabulary's logits are 0.5 MB).  x: x_len >= cols floats in host
 * memory; token, prob, kept: one each, the last two may be NULL.  The checks of
 * both calls apply; a weight of 0 rows or more than 4194304 -> ARG. */
int32_t gollek_hip_next_token(gollek_hip_weight *lm_head, const float *x, int64_t x_len, float temperature,
                              int32_t top_k, float top_p, float min_p, float u, int32_t *token, float *prob,
                              int32_t *kept, char *err, size_t err_len);

/* ---- between the products of a decoder layer ------------------------------- */

/* Element types of these calls: F32, F16 and BF16 (ggml type ids 0, 1, 30); any
 * other -> UNSUPPORTED.  Computed in fp32 and rounded once (to nearest).  Device
 * forms are asynchronous on the caller's stream, allocate nothing and can be
 * captured into a graph; their arrays are aligned to their elements (else ARG), and
 * what a call writes must not share memory with what it reads or with its other
 * results, unless said otherwise (-> ARG).  A stride is the number of elements
 * between two rows (0: packed).  The reference's GGUF path leaves these to its Java
 * runner; none of them replaces an entry of it. */

#define GOLLEK_HIP_NORM_RMS 0   /* N(v) = v / sqrt(mean(v^2) + eps) */
#define GOLLEK_HIP_NORM_LAYER 1 /* N(v) = (v - mean(v)) / sqrt(mean((v - mean(v))^2) + eps) */

/* The norms around a block, row by row (rows x cols):
 *   b = post_weight ? N(x) * post_weight : x
 *   h = residual + scale * gate * b               -> hidden, of hidden_type
 *   y = N(h) * weight + bias                      -> y, of y_type
 * with N by `kind` and h unrounded in N(h).  post_weight, gate, weight, bias: cols
 * floats; residual: of hidden_type; NULL: no first norm, gate 1, residual 0, weight 1,
 * bias 0; hidden or y may be NULL (not both).  rows up to 2^31 - 1, cols in
 * [1, 65536], a finite scale, eps >= 0 and finite: else ARG.  hidden may be x or the
 * residual itself, y may be x or the residual (the same address, type size and
 * stride).  The sum of a row's squares is fp32's: it has to stay below 3.4e38, a root
 * mean square below 1.8e19 / sqrt(cols) (2.8e17 at 4096, 7.2e16 at 65536), else the
 * norm is 0.  With eps 0 a row of zeros divides 0 by 0 (NaN), and so small a row that
 * its squares are 0 (elements below 1e-23) divides by 0 (infinities).
 * The host form takes packed rows and copies them up (synchronous). */
int32_t gollek_hip_norm(const void *x, int32_t x_type, int64_t rows, int64_t cols, const float *post_weight,
                        const float *gate, float scale, const void *residual, void *hidden, int32_t hidden_type,
                        const float *weight, const float *bias, int32_t kind, float eps, void *y, int32_t y_type,
                        char *err, size_t err_len);
int32_t gollek_hip_norm_device(const void *x, int32_t x_type, int64_t rows, int64_t cols, int64_t x_stride,
                               const float *post_weight, const float *gate, float scale, const void *residual,
                               int64_t residual_stride, void *hidden, int32_t hidden_type, int64_t hidden_stride,
                               const float *weight, const float *bias, int32_t kind, float eps, void *y,
                               int32_t y_type, int64_t y_stride, void *stream, char *err, size_t err_len);

/* Rotary positions: which elements of a head's first `dims` make a pair. */
#define GOLLEK_HIP_ROPE_HALF 0        /* i and i + dims / 2 */
#define GOLLEK_HIP_ROPE_INTERLEAVED 1 /* 2 i and 2 i + 1 */
/* How their frequencies f_i = base^(-2 i / dims) are scaled for long contexts. */
#define GOLLEK_HIP_ROPE_NONE 0
#define GOLLEK_HIP_ROPE_LINEAR 1 /* f / factor */
#define GOLLEK_HIP_ROPE_YARN 2   /* f / factor where a pair turns fewer than `low` times in original_context, f where more
                                  * than `high` times, mixed by a ramp over the pairs between; magnitude 0.1 ln(factor) + 1 */
#define GOLLEK_HIP_ROPE_LLAMA3 3 /* the same borders, mixed by the number of turns; magnitude 1 */

/* Opaque table of a model's rotary frequencies, on the device that was current.  It
 * must outlive every call that takes it, and every captured graph that holds one: a
 * replay reads the table again. */
typedef struct gollek_hip_rope gollek_hip_rope;

/* Frequencies (radians a position, dims / 2 floats) and magnitude (one float) that
 * a table of these arguments has; either may be NULL; needs no GPU.  Pair i of a head
 * turns by position * f_i and is multiplied by the magnitude; magnitude 0 stands for
 * the scaling's own (1, or YARN's).  factors: dims / 2 floats that divide the
 * frequencies first (a GGUF file's rope_freqs.weight), or NULL.  dims even in
 * [2, 256], base > 1, and where the scaling uses them factor > 0, original_context > 0
 * and 0 < low < high; everything finite, magnitude >= 0, factors > 0: else ARG.  The
 * table itself is in 64 bits: a position of 2^31 keeps its angle. */
int32_t gollek_hip_rope_frequencies(int64_t dims, float base, int32_t scaling, float factor, float original_context,
                                    float low, float high, float magnitude, const float *factors, float *frequencies,
                                    float *resulting_magnitude, char *err, size_t err_len);
/* NULL on failure.  An unknown layout -> ARG. */
gollek_hip_rope *gollek_hip_rope_create(int32_t layout, int64_t dims, float base, int32_t scaling, float factor,
                                        float original_context, float low, float high, float magnitude,
                                        const float *factors, char *err, size_t err_len);
/* Waits for the device's work first; captures that go on are left alone.  NULL is a no-op. */
void gollek_hip_rope_free(gollek_hip_rope *rope);

/* out = x (tokens x heads x head_dim) with every head's first dims elements rotated
 * to its token's position, the others as they are; out of x's type, may be x itself
 * (with its stride).  head_dim even in [dims, 256], heads in [1, 65535], tokens up to
 * 2^31 - 1: else ARG.  The host form takes packed rows and copies them up. */
int32_t gollek_hip_rope_apply(const gollek_hip_rope *rope, const void *x, int32_t type, int64_t tokens, int64_t heads,
                              int64_t head_dim, const int32_t *positions, void *out, char *err, size_t err_len);
int32_t gollek_hip_rope_apply_device(const gollek_hip_rope *rope, const void *x, int32_t type, int64_t tokens,
                                     int64_t heads, int64_t head_dim, int64_t x_stride, const int32_t *positions,
                                     void *out, int64_t out_stride, void *stream, char *err, size_t err_len);

/* Opaque paged cache of keys and values: a view of two device arrays that the
 * caller keeps, each (pages x kv_heads x page_size x head_dim) of `type`, F16 or BF16. */
typedef struct gollek_hip_kv_cache gollek_hip_kv_cache;

/* page_size a power of two in [16, 65536], head_dim a multiple of 8 in [8, 256],
 * kv_heads in [1, 65535], pages in [1, 2^31 - 1], k and v 16-byte aligned and apart:
 * else ARG; another type -> UNSUPPORTED.  NULL on failure. */
gollek_hip_kv_cache *gollek_hip_kv_cache_wrap_device(int32_t type, void *k, void *v, int64_t pages, int64_t page_size,
                                                     int64_t kv_heads, int64_t head_dim, char *err, size_t err_len);
/* Frees the handle, not the arrays, which calls and captured graphs go on using.  NULL is
 * a no-op. */
void gollek_hip_kv_cache_free(gollek_hip_kv_cache *cache);

/* Appends new tokens to a cache, and makes their queries ready for it:
 *   k, v (tokens x kv_heads x head_dim of `type`): k by k_norm and rope -> the cache
 *     at the token's place, v as it is;
 *   q (tokens x q_heads x head_dim of `type`, NULL with q_heads 0): by q_norm and
 *     rope -> q_out, of the cache's type.
 * q_norm, k_norm (head_dim floats, NULL: none): RMS norms of each head before it
 * turns; rope NULL: no rotation.  The place of token t is position positions[t] of
 * sequence sequence[t] (NULL: t), in page page_table[sequence * max_pages +
 * position / page_size].  A token whose position is below 0, or whose sequence is
 * outside [0, sequences), is padding: nothing of it is written.  Where the position
 * is past the table (max_pages * page_size) or the page outside [0, pages), k and v
 * are dropped.  Two tokens of a call must not have one place: which of them stays is
 * not determined.  q_out may be q itself where the types have one size (and with its
 * stride).  tokens up to 2^31 - 1, q_heads in [0, 65535], max_pages >= 1 with
 * max_pages * page_size < 2^31, rope's dims at most head_dim, rope on the cache's
 * device: else ARG. */
int32_t gollek_hip_kv_append_device(const gollek_hip_kv_cache *cache, const gollek_hip_rope *rope, const void *k,
                                    int64_t k_stride, const void *v, int64_t v_stride, const void *q, int64_t q_heads,
                                    int64_t q_stride, int32_t type, int64_t tokens, const float *q_norm,
                                    const float *k_norm, float eps, const int32_t *positions, const int32_t *sequence,
                                    const int32_t *page_table, int64_t sequences, int64_t max_pages, void *q_out,
                                    int64_t q_out_stride, void *stream, char *err, size_t err_len);

/* Attention of one new token a sequence over the cache.  q (sequences x q_heads x
 * head_dim of the cache's type, as gollek_hip_kv_append_device leaves it); q_heads a
 * multiple of kv_heads, whose q_heads / kv_heads neighbours share keys and values:
 *   s_j = scale * q . k_j,  capped: softcap * tanh(s_j / softcap) (softcap 0: not)
 *   out = sum_j exp(s_j) v_j / (sum_j exp(s_j) + exp(sinks[head]))   (sinks NULL: no such term)
 * over the last `window` (0: all) of the first lengths[sequence] tokens, -> out
 * (sequences x q_heads x head_dim of out_type).  A length past the table counts as
 * the table's, one below 1 as 0; a token whose page is outside [0, pages) is not
 * there; a row without any token (or with every s_j -inf) is 0.  Nothing behind a sequence's length or before
 * its window changes a result, whatever it holds.  An infinite value among the others
 * makes its dim's results infinite whatever its weight, a NaN or two infinities of other
 * signs make them NaN.  Several new tokens of one
 * sequence are rows of their own, with equal page_table rows and growing lengths.
 * Weights multiply the values with 24 bits (BF16 caches) or 22 (F16); scores and sums are
 * fp32's: scores past 2.3e38 and values that add up past 3.4e38 overflow.
 * Results depend in their last bits on the batch (its rows, lengths and table width set
 * how the sums are split), not on timing.  sequences and q_heads in [0, 65535] and
 * [1, 65535], sequences * q_heads < 2^24, max_pages as above, scale in [-1e15, 1e15],
 * softcap 0 or in [1e-15, 1e15], window >= 0, workspace (256-byte aligned; calls sharing it must not
 * overlap) of at least gollek_hip_attention_workspace_bytes: else ARG. */
int32_t gollek_hip_attention_device(const gollek_hip_kv_cache *cache, const void *q, int64_t q_stride,
                                    int64_t sequences, int64_t q_heads, const int32_t *lengths,
                                    const int32_t *page_table, int64_t max_pages, float scale, float softcap,
                                    int64_t window, const float *sinks, void *out, int32_t out_type,
                                    int64_t out_stride, void *workspace, int64_t workspace_bytes, void *stream,
                                    char *err, size_t err_len);
/* Device workspace bytes that call needs (-1: out of range).  They never fall as
 * sequences or max_pages rise. */
int64_t gollek_hip_attention_workspace_bytes(const gollek_hip_kv_cache *cache, int64_t sequences, int64_t q_heads,
                                             int64_t max_pages);

/* ---- GGUF files --------------------------------------------------------- */
/* GC/ = runner/gguf/gollek-gguf-core/src/main/java/tech/kayys/gollek/gguf/. */

/* Opaque parsed GGUF file (a read-only mapping of it plus its tensor table). */
typedef struct gollek_hip_gguf gollek_hip_gguf;

/* Maps `path` read-only and parses the header, the metadata (skipped, except
 * general.alignment, default 32) and the tensor infos; needs no GPU.
 * Replaces GC/loader/GGUFReader.java:28-37 (open + mmap) with
 * GC/loader/GGUFParser.java:17-105 (parse).  Returns NULL with the status
 * (gollek_hip_last_status) and message set: bad magic -> ARG "Not a valid
 * GGUF file"; a metadata type outside 0..12 -> UNSUPPORTED "Unsupported GGUF
 * KV type: N at pos P"; a tensor type without a GGUF block layout or an
 * element count that is not a multiple of its block -> UNSUPPORTED
 * "Unsupported or misaligned GGUF tensor type T with N element(s)"; a
 * truncated file, a negative or oversized length or count, more than 8
 * dimensions, a non-numeric or non-positive general.alignment -> ARG. */
gollek_hip_gguf *gollek_hip_gguf_open(const char *path, char *err, size_t err_len);

/* Unmaps the file and frees its upload buffers.  Weight handles uploaded from
 * it stay valid.  NULL is a no-op. */
void gollek_hip_gguf_close(gollek_hip_gguf *file);

/* Header facts: format version, tensor and metadata counts, the alignment
 * used, the absolute offset of the tensor data (GGUFModel.dataStart,
 * GC/loader/GGUFParser.java:57-62) and the file size.  Any pointer may be NULL. */
int32_t gollek_hip_gguf_info(const gollek_hip_gguf *file, int32_t *version, int64_t *n_tensors,
                             int64_t *n_kv, int64_t *alignment, int64_t *data_start,
                             int64_t *file_bytes);

/* Tensor `index` in file order (GC/loader/GGUFTensorInfo.java:8-14): name
 * (NUL-terminated, truncated to name_len - 1), ggml type id, dimension count,
 * dims[0..7] (dims[0] = the contiguous one; unused entries 1), offset from
 * the data start and size in bytes.  Index out of range -> ARG.  Output
 * pointers may be NULL. */
int32_t gollek_hip_gguf_tensor(const gollek_hip_gguf *file, int64_t index, char *name,
                               size_t name_len, int32_t *type_id, int32_t *n_dims, int64_t *dims,
                               int64_t *offset, int64_t *size_bytes);

/* Index of the first tensor named `name` (GGUFModel.tensors lookup by name),
 * or -1. */
int64_t gollek_hip_gguf_find(const gollek_hip_gguf *file, const char *name);

/* Copies tensor `index` to a new device weight handle on the current device
 * (rows = product of dims[1..], cols = dims[0]), through pinned staging
 * buffers the file object keeps.  Replaces the byte slice of
 * GC/runtime/GgufTensorData.java:97-104 followed by gollek_hip_weight_upload:
 * bytes outside the file -> ARG "Tensor data range is outside model segment:
 * NAME"; then the validation of gollek_hip_weight_upload (types other than
 * Q4_0 / Q8_0 / Q4_K / Q5_K / Q6_K -> UNSUPPORTED).  Free the handle with
 * gollek_hip_weight_free.  Thread-safe; uploads from one file object
 * serialise on its staging buffers. */
gollek_hip_weight *gollek_hip_gguf_upload(gollek_hip_gguf *file, int64_t index, char *err,
                                          size_t err_len);

#ifdef __cplusplus
}
#endif
#endif /* GOLLEK_HIP_H */
