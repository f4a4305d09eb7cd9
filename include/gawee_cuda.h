/*
 * libgawee_cuda — B200 (sm_100a) backend for compiled inference of a
 * gawee-dialect `forward` function.
 *
 * It replaces the CPU code generation of `gawee-opt --gawee-to-llvm`
 * (middle/mlir/tools/gawee-opt.cpp:120-184) and the AOT launcher/runtime
 * (back/gawee_aot.cpp:174-291, back/runtime_support.h) for the same graph:
 * the graph text that `gawee-onnx-translate` prints is planned into a static
 * sequence of CUDA kernels, weights stay resident on the GPU, and each
 * forward replays the sequence.
 *
 * Conventions
 *   - Arguments are the `forward` arguments in order: graph inputs, then the
 *     float initializers (middle/mlir/lib/Emit/ONNXMLIREmitter.cpp:2932-2975).
 *   - Host buffers are dense C-order arrays of the argument's static shape;
 *     the caller owns them.  Boolean (i1) tensors use one byte per element.
 *   - No exception crosses this interface; every call returns a gawee_status.
 *     gawee_last_error() returns the message of the last failure on a context.
 *   - One context per device.  Calls on one context must be serialised by
 *     the caller; contexts on different devices may be used from different
 *     host threads.
 *   - `stream` arguments are cudaStream_t values passed as void* (NULL means
 *     the context's own stream).
 */
#ifndef GAWEE_CUDA_H
#define GAWEE_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef int gawee_status;
enum {
  GAWEE_OK = 0,
  GAWEE_ERR_INVALID = 1,      /* bad argument, index, size or state */
  GAWEE_ERR_PARSE = 2,        /* the MLIR text could not be parsed */
  GAWEE_ERR_UNSUPPORTED = 3,  /* an op or shape the backend does not implement */
  GAWEE_ERR_CUDA = 4,         /* a CUDA runtime error */
  GAWEE_ERR_OOM = 5,          /* device allocation failed */
  GAWEE_ERR_DEVICE = 6,       /* a kernel reported an error (e.g. gather index out of range) */
  GAWEE_ERR_NCCL = 7          /* a NCCL call failed */
};

/* Element types (numbering shared with the planner). */
enum {
  GAWEE_F32 = 0,
  GAWEE_F64 = 1,
  GAWEE_F16 = 2,
  GAWEE_I64 = 3,
  GAWEE_I32 = 4,
  GAWEE_I1 = 5,
  GAWEE_BF16 = 7 /* paged key/value cache only; 6 is taken by the planner */
};

typedef struct gawee_ctx gawee_ctx;

/* Plan the function `entry` (NULL = "forward") of MLIR module text for
 * `device`.  Replaces `gawee-opt --gawee-to-llvm` + `gawee-aot build`
 * (back/gawee_aot.cpp:325-366): parsing, fusion, memory planning and device
 * allocation happen here, once. */
gawee_status gawee_create(const char* mlir_text, const char* entry, int device, gawee_ctx** out);

/* Same, reading the MLIR text from a file. */
gawee_status gawee_create_from_file(const char* mlir_path, const char* entry, int device, gawee_ctx** out);

void gawee_destroy(gawee_ctx* ctx);

/* Copies the last error message (NUL-terminated, truncated to n). */
gawee_status gawee_last_error(const gawee_ctx* ctx, char* buf, size_t n);

/* Signature of `forward`: counts, dtypes and static shapes (shape needs room
 * for `rank` values; rank <= 8).  Mirrors parseFuncSignature
 * (back/gawee_aot.cpp:104-144). */
int gawee_num_args(const gawee_ctx* ctx);
int gawee_num_outputs(const gawee_ctx* ctx);
gawee_status gawee_arg_info(const gawee_ctx* ctx, int i, int* dtype, int* rank, int64_t* shape);
gawee_status gawee_output_info(const gawee_ctx* ctx, int i, int* dtype, int* rank, int64_t* shape);

/* Stage argument i from host memory (asynchronous on `stream`; pinned host
 * memory gives true overlap).  Replaces loadNpy + makeDescriptor per argument
 * (back/gawee_aot.cpp:241-249).  Weights that are re-staged are re-packed on
 * the next forward; otherwise packed weights stay resident. */
gawee_status gawee_set_arg(gawee_ctx* ctx, int i, const void* host, size_t bytes, void* stream);

/* Stage argument i from device memory on the context's device. */
gawee_status gawee_set_arg_device(gawee_ctx* ctx, int i, const void* dev, size_t bytes, void* stream);

/* Device pointer of argument i, in the context's memory until it is destroyed: for
 * the pages of a gawee.paged_attention op, which the forward updates in place and
 * the gawee_kv calls below can fill and evict from.  An argument that is a
 * packed weight is written with gawee_set_arg instead. */
gawee_status gawee_arg_device_ptr(gawee_ctx* ctx, int i, void** ptr);

/* Whether the forward writes argument i, as it does the pages of a
 * gawee.paged_attention op: 1 or 0, -1 for an index out of range. */
int gawee_arg_in_place(const gawee_ctx* ctx, int i);

/* Copy an argument that the forward writes back to host memory (asynchronous on `stream`). */
gawee_status gawee_get_arg(gawee_ctx* ctx, int i, void* host, size_t bytes, void* stream);

/* Enqueue one forward on `stream`.  Replaces the call of
 * _mlir_ciface_forward (back/gawee_aot.cpp:263-274).  Asynchronous. */
gawee_status gawee_forward(gawee_ctx* ctx, void* stream);

/* Copy output i to host memory (asynchronous on `stream`).  Replaces
 * saveReturnedMemRef (back/runtime_support.h:272-277). */
gawee_status gawee_get_output(gawee_ctx* ctx, int i, void* host, size_t bytes, void* stream);

/* Device pointer of output i (valid until the next forward). */
gawee_status gawee_output_device_ptr(gawee_ctx* ctx, int i, void** ptr);

/* Wait for `stream` and check the device status word: returns
 * GAWEE_ERR_DEVICE if a kernel flagged an error since the last check.  With
 * ctx NULL it checks the status word of gawee_matmul_f32_noalloc on the
 * current device instead (message via gawee_last_error(NULL, ...)). */
gawee_status gawee_synchronize(gawee_ctx* ctx, void* stream);

/* Capture the forward sequence into a CUDA graph on the next forward
 * (enabled = 1, the default) or launch kernels one by one (0). */
gawee_status gawee_set_graph_mode(gawee_ctx* ctx, int enabled);

/* Arithmetic of the tensor-core contractions (convolutions, GEMMs, fused
 * attention).  The reference computes in fp32 on the CPU; there is no
 * reference counterpart to this call.
 *   GAWEE_PRECISION_FP32 (default): each product from three TF32 products of
 *     the operands' high parts and remainders (hi*hi + hi*lo + lo*hi), fp32
 *     accumulation with round-to-nearest promotion every 64 k: parity with
 *     the fp32 reference at its own tolerances.
 *   GAWEE_PRECISION_TF32: one TF32 product of the truncated operands (10
 *     explicit mantissa bits each), same accumulation: |error| <= 2^-9 *
 *     sum |a_k * b_k| per output plus the accumulation term; not a parity mode.
 *   GAWEE_PRECISION_BF16: contractions on the TMA kernel take one bf16
 *     product (both operands rounded to nearest bf16, 8 significant bits,
 *     relative error <= 2^-9 each), same fp32 accumulation: |error| <=
 *     2^-8 * sum |a_k * b_k| plus the accumulation term; the other
 *     tensor-core kernels (the gather kernel, fused attention) run single-pass
 *     TF32.  The first switch to it allocates a bf16 copy of those
 *     contractions' B operands (half the size of one packed plane).
 * GAWEE_PRECISION=tf32 or bf16 in the environment selects the mode at
 * gawee_create.  Changing the mode drops the captured CUDA graph (it is
 * captured again on the next forward); call it between forwards, with no
 * forward in flight. */
enum { GAWEE_PRECISION_FP32 = 0, GAWEE_PRECISION_TF32 = 1, GAWEE_PRECISION_BF16 = 2 };
gawee_status gawee_set_precision(gawee_ctx* ctx, int mode);
int gawee_precision(const gawee_ctx* ctx); /* the current mode, -1 for NULL */

/* Kernel i of the per-forward sequence: name (fused ops joined by '+'),
 * whether it is a tensor-core contraction, and its algorithmic FLOPs
 * (2*M*N*K with the unpadded K; 0 for other kernels). */
gawee_status gawee_op_info(const gawee_ctx* ctx, int i, char* name, size_t n, int* is_tc, double* flops);

/* Run one forward eagerly with a CUDA event between every kernel and write
 * each kernel's device time in milliseconds to ms[0..gawee_num_kernels-1].
 * Synchronous. */
gawee_status gawee_profile_forward(gawee_ctx* ctx, void* stream, float* ms, int n);

/* Plan without a device: parse and plan `entry` of MLIR text and write the
 * plan summary (or the error message) into buf.  No CUDA call is made. */
gawee_status gawee_plan_text(const char* mlir_text, const char* entry, char* buf, size_t n);

/* Planned main-sequence steps of one forward (the index space of
 * gawee_op_info / gawee_profile_forward) and a human-readable plan summary.
 * gawee_num_launches counts the kernel launches of one forward: a step whose
 * contraction is split along k adds a reduce kernel. */
int gawee_num_kernels(const gawee_ctx* ctx);
int gawee_num_launches(const gawee_ctx* ctx);
gawee_status gawee_plan_summary(const gawee_ctx* ctx, char* buf, size_t n);

/* ---------------------------------------------------------------------------
 * _mlir_ciface_forward compatibility.
 *
 * The reference launcher calls
 *   void _mlir_ciface_forward(MemRefDescriptor<T,R>* result, MemRefDescriptor<Ti,Ri>* arg0, ...)
 * (back/gawee_aot.cpp:174-195, struct at back/runtime_support.h:21-28).
 * gawee_ciface_forward takes the same descriptors as an array: it stages every
 * argument, runs one forward, waits, and writes the single result into a
 * malloc'ed buffer described by `result` (the callee allocates, as the
 * reference's lowered code does).  A memref descriptor is
 *   { T* allocated; T* aligned; int64_t offset; int64_t sizes[R]; int64_t strides[R]; }
 * and must describe a dense C-order array.  An argument that the forward
 * writes (gawee_arg_in_place: the pages of a gawee.paged_attention op) is copied back
 * into the caller's array, so that the next call has the rows which this one stored.
 * A loop that keeps its pages on the device uses gawee_set_arg for what changes, and gawee_forward.
 * ------------------------------------------------------------------------- */
gawee_status gawee_ciface_forward(gawee_ctx* ctx, void* result_desc, void* const* arg_descs, int nargs);

/* Entry point for code produced by the `--gawee-to-cuda` pipeline: the
 * lowered module keeps the gawee-level `forward` text as a global string and
 * its `_mlir_ciface_forward` calls this.  The first call on a thread plans the
 * text for `device` and caches the context (keyed by the string's address);
 * later calls reuse it.  Semantics as gawee_ciface_forward; on failure the
 * message is read with gawee_last_error(NULL, ...). */
gawee_status gawee_embedded_forward(const char* mlir_text, int device, void* result_desc, void* const* arg_descs,
                                    int nargs);

/* ---------------------------------------------------------------------------
 * Allocation-free matrix product (no counterpart in the reference).
 *
 * C[m][n] = A[m][k] . B[k][n], fp32 row-major device arrays owned by the
 * caller, computed on the tensor-core kernel with split-precision TF32
 * (the same arithmetic as gawee.matmul in a planned graph), enqueued on
 * `stream`.  For callers that cannot allocate device memory when they need
 * the product: a host framework whose own caching allocator owns the device
 * memory (an allocation behind its back can fail or fragment its pool), a
 * caller working within a fixed memory budget, or an error-recovery path
 * after an allocation has already failed; cudaMalloc and cudaFree can also
 * wait for the whole device.  It calls no cudaMalloc/cudaFree and no
 * allocating library routine: the packed TF32 planes of B use a 16 MiB array
 * in the library's static device memory, which every GPU that loads the
 * library holds until the process exits.
 *   - Limits: k a multiple of 4, A 16-byte aligned, n * k <= 2,097,152
 *     (two planes of n x k floats in 16 MiB); larger shapes return
 *     GAWEE_ERR_INVALID with a message for gawee_last_error(NULL, ...).
 *   - The first call on a device looks up the device addresses of the array
 *     and of a status word (cudaGetSymbolAddress); make that first call
 *     before any stream capture.
 *   - Every call shares the one array: calls that overlap on the GPU (on
 *     different streams, or from several threads) race.  Each call rewrites
 *     all of the scratch it reads, so nothing needs clearing between calls.
 *   - Errors inside the kernel (a bounded wait that gave up, leaving C
 *     partly written) are recorded in the shared status word:
 *     gawee_synchronize(NULL, stream) waits for `stream`, then returns
 *     GAWEE_ERR_DEVICE and clears the word if any call since the last check
 *     reported one.
 * ------------------------------------------------------------------------- */
gawee_status gawee_matmul_f32_noalloc(const float* a, const float* b, float* c, int64_t m, int64_t n, int64_t k,
                                      void* stream);

/* ---------------------------------------------------------------------------
 * Paged key/value cache (no counterpart in the reference, whose decode step
 * concatenates the cache anew for each token and is compiled for one length).
 *
 * The keys and values of many sequences lie in pages of page_size rows, two
 * arrays [num_pages][kv_heads][page_size][head_dim] of f32, f16 or bf16 that
 * the caller owns (one pair per layer).  A block table, int32 [batch][columns]
 * on the device, names each sequence's pages in order: row i of sequence b is
 * slot i % page_size of page table[b][i / page_size].  Columns behind a
 * sequence's last row are never read.  Lengths and tables are read on the
 * device when the call runs, so that one captured call serves every step.
 *
 * In a graph, gawee.paged_attention(q, k, v, k_pages, v_pages, block_table,
 * lengths) <{scale}> is gawee_kv_attend with k and v: f32, the table and lengths i32,
 * the pages two function arguments that nothing else uses; they live in the context and
 * keep the stored rows from one forward to the next, until gawee_set_arg replaces them.
 * The calls that stage every argument from host memory (gawee_ciface_forward,
 * gawee_embedded_forward, Model.run in Python) copy the pages back after the forward;
 * the file contract of gawee-cuda-runner has no place for them.
 *
 * A gawee_kv handle holds the shapes and the scratch memory, allocated once;
 * one handle serves any number of layers.
 *   - Every pointer is device memory of the handle's device; activations (q,
 *     out, k, v) are of one type, f32, f16 or bf16, whatever the pages' type.
 *     Pages are 16-byte aligned, and so is the distance between two pages.
 *     Arrays of a call do not overlap unless a call says so.
 *   - Calls enqueue on `stream` (NULL: the device's default stream), do not
 *     wait, allocate nothing and can be captured into a graph.  They leave the
 *     calling thread's current device as it was.
 *   - Calls on one handle share its scratch: they are ordered by the caller,
 *     by one stream or by events; replays of graphs that hold them too.  Calls
 *     that may run at the same time take a handle each.  (Nothing of one call
 *     stays in the scratch for the next: calls that overlap against this rule
 *     spoil their own results, and no later ones.)
 *   - What a call reads (lengths, tables, positions, weights) is not written by
 *     others while it runs.
 *   - A bad argument is refused with GAWEE_ERR_INVALID before anything is
 *     enqueued; the message is read with gawee_last_error(NULL, ...).
 *   - What only the device can see (a table entry that names no page, a length
 *     beyond the table) is recorded in the handle, and gawee_kv_synchronize
 *     returns GAWEE_ERR_DEVICE; memory outside the arrays is not touched.
 * ------------------------------------------------------------------------- */
typedef struct gawee_kv gawee_kv;

typedef struct {
  int dtype;           /* of the pages: GAWEE_F32, GAWEE_F16 or GAWEE_BF16 */
  int heads;           /* query heads, a multiple of kv_heads, up to 4096 */
  int kv_heads;        /* query head h reads key/value head h / (heads / kv_heads) */
  int head_dim;        /* a multiple of 8, up to 256 */
  int page_size;       /* rows of a page, up to 65536 */
  int64_t num_pages;
  int64_t page_stride; /* elements between pages; 0: kv_heads * page_size * head_dim */
  int max_batch;       /* sequences of a call at most, up to 65535 */
  int max_pages;       /* columns of a block table at most */
  int weights;         /* nonzero: gawee_kv_attend may return attention weights (scratch of
                          max_batch * heads * max_pages * page_size floats) */
} gawee_kv_desc;

/* device -1: a handle without a device, whose calls check their arguments and
 * then return GAWEE_ERR_CUDA (as gawee_plan_text plans without one). */
gawee_status gawee_kv_create(const gawee_kv_desc* desc, int device, gawee_kv** out);
void gawee_kv_destroy(gawee_kv* kv); /* waits for the device's work first */

typedef struct {
  void* k_pages;
  void* v_pages;
  const void* k; /* new rows [tokens][kv_heads][head_dim], stored rounded to nearest in the pages' type */
  const void* v;
  int dtype;        /* of k and v */
  int64_t k_stride; /* elements between tokens; a column slice of a wider projection is fine */
  int64_t v_stride;
  int64_t tokens;
  const int32_t* sequences; /* [tokens]: row of the block table; NULL: token t is of sequence t */
  const int32_t* positions; /* [tokens]: row within the sequence */
  const int32_t* block_table;
  int64_t table_stride; /* elements between rows */
  int table_cols;
  int batch; /* rows of the block table */
} gawee_kv_append_args;

/* Write the rows of new tokens (a prompt, or one token per sequence) into the
 * pages.  Tokens with a negative sequence or position are left out.  Two
 * tokens of one call that name the same row leave a mixture of the two there. */
gawee_status gawee_kv_append(gawee_kv* kv, const gawee_kv_append_args* args, void* stream);

typedef struct {
  void* k_pages; /* written only where k and v are given */
  void* v_pages;
  const void* q; /* [batch][heads][head_dim] */
  void* out;     /* [batch][heads][head_dim] */
  int dtype;     /* of q, out, k and v */
  int64_t q_stride; /* elements between sequences */
  int64_t out_stride;
  int batch;
  float scale; /* of the scores: 1 / sqrt(head_dim) as a rule */
  const int32_t* block_table;
  int64_t table_stride;
  int table_cols;
  const int32_t* lengths; /* [batch]: cached rows, the new token's own among them */
  const void* k; /* optional, with v: [batch][kv_heads][head_dim], the new token's rows */
  const void* v;
  int64_t k_stride;
  int64_t v_stride;
  const float* mask; /* optional: [batch][mask_cols], added to the scaled scores */
  int64_t mask_stride;
  int64_t mask_cols;
  const float* weights; /* optional: [batch][kv_heads][weights_cols], accumulated attention weights */
  int64_t weights_stride;       /* elements between heads */
  int64_t weights_batch_stride; /* elements between sequences */
  float* weights_out;           /* the same after this step; may be `weights` itself */
  int64_t weights_out_stride;
  int64_t weights_out_batch_stride;
  int64_t weights_cols;
} gawee_kv_attend_args;

/* Attention of one new token per sequence over its rows 0 .. length - 1:
 *   out[b][h] = sum_i p_i V_i,  p = softmax_i(scale * (q[b][h] . K_i) + mask[b][i]),
 * with fp32 scores, maxima and sums.  Where pages and activations are of one 16-bit
 * type, the weights may enter the products with V as two terms of that type: off by 2^-16
 * relatively in bf16, in f16 by 2^-21 or by 2^-40 of the largest weight,
 * whichever is more; otherwise they are fp32.  With k and v, they are first stored as
 * row length - 1 (rounded to the pages' type, and attended as stored); the
 * page of that row then belongs to this sequence alone.  With weights_out,
 * each row's weights, summed over the query heads that share its key/value
 * head, are added: weights_out = weights + sum_h p_h (weights NULL: zeros);
 * columns from length on are not touched.
 *   - A mask value of -inf takes the row out, whatever its K and V or the query hold.  Other
 *     values are added as they are: a mask of the lowest finite value is one.
 *     A sequence of length 0, or whose rows are all taken out, gives zeros.
 *     A mask value of +inf or NaN gives NaN.
 *   - A negative length marks a batch row without a sequence: its rows of out,
 *     weights_out and the pages are left as they were.
 *   - The same call gives the same bits: partial sums are joined in a fixed
 *     order, which depends on the shapes and the lengths of the batch. */
gawee_status gawee_kv_attend(gawee_kv* kv, const gawee_kv_attend_args* args, void* stream);

typedef struct {
  void* k_pages;
  void* v_pages;
  const float* weights; /* [batch][kv_heads][weights_cols], as accumulated by gawee_kv_attend */
  int64_t weights_stride;
  int64_t weights_batch_stride;
  float* weights_out; /* of the kept rows, at their new places; may be `weights` itself */
  int64_t weights_out_stride;
  int64_t weights_out_batch_stride;
  int64_t weights_cols;
  int batch;
  const int32_t* block_table;
  int64_t table_stride;
  int table_cols;
  const int32_t* to_table; /* NULL: in place; else [batch][to_cols], the pages that receive the kept rows */
  int64_t to_stride;
  int to_cols;
  const int32_t* lengths;
  int32_t* lengths_out; /* may be `lengths` itself */
  int budget;           /* rows that a sequence keeps at most: at least 1, below 2^31 - 2^24 */
  int recent;           /* of these, the last rows that always stay, 0 .. budget */
  int32_t* kept;        /* [batch][kv_heads][budget]: earlier positions of the kept rows, ascending; -1 behind them */
} gawee_kv_evict_args;

/* Cut sequences longer than `budget` down to it.  Each key/value head keeps
 * the last `recent` rows and, of the others, the budget - recent of greatest
 * weight (equal weights: the lowest position; NaN below every number).  Kept rows move, in
 * order, to rows 0 .. budget - 1; their weights too, and weights_out from there to
 * the old length becomes 0; lengths_out = min(length, budget).  Sequences
 * within the budget keep every row.
 *   - In place, a sequence's pages belong to it alone; those behind the budget
 *     are free afterwards.  With to_table, all kept rows are copied into its
 *     pages, which are no sequence's pages in block_table: pages shared between sequences stay whole.
 *   - A negative length marks a batch row without a sequence: its kept is -1, its
 *     length is passed on, nothing else is touched. */
gawee_status gawee_kv_evict(gawee_kv* kv, const gawee_kv_evict_args* args, void* stream);

/* Wait for `stream` and check the handle's status word: GAWEE_ERR_DEVICE if a
 * call flagged an error since the last check. */
gawee_status gawee_kv_synchronize(gawee_kv* kv, void* stream);

/* Diagnostic: the tensor cores' TF32 rate on `device`, measured now (one CTA
 * per SM issuing back-to-back M = 128, N = 128, K = 8 tcgen05 TF32 MMAs with
 * both operands in shared memory, timed with CUDA events; about 5 ms).  The
 * fp32 mode issues three such products per multiply-add, so a third of
 * *tflops is its tensor ceiling.  No reference counterpart. */
gawee_status gawee_probe_tf32_mma(int device, double* tflops);

/* ---------------------------------------------------------------------------
 * Data parallelism: batch sharding with replicated weights (one process or
 * thread per GPU).  The only collective is the gather of each rank's output
 * rows to rank 0 over NCCL.
 * ------------------------------------------------------------------------- */
#define GAWEE_NCCL_ID_BYTES 128

/* Fill `id` (GAWEE_NCCL_ID_BYTES) on rank 0; share it with the other ranks. */
gawee_status gawee_dp_unique_id(void* id);

/* Join a communicator of `world` ranks on the context's device.  Collective:
 * the ranks also exchange their output sizes (shards may differ by a row,
 * e.g. 5 rows over 2 ranks as 3 + 2). */
gawee_status gawee_dp_init(gawee_ctx* ctx, int world, int rank, const void* id);

/* Bytes of output i summed over every rank: the size of rank 0's
 * destination buffer for gawee_dp_gather_output. */
gawee_status gawee_dp_output_bytes(gawee_ctx* ctx, int i, size_t* total);

/* Gather output i of every rank, in rank order, into `dst` on rank 0 (a
 * device buffer of gawee_dp_output_bytes bytes; ignored on other ranks).
 * Each rank contributes its own output size, as exchanged at init.
 * Collective: every rank calls it, in the same order. */
gawee_status gawee_dp_gather_output(gawee_ctx* ctx, int i, void* dst, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* GAWEE_CUDA_H */
