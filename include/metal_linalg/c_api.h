/* The C ABI of the B200 build of metal-linalg's QR path: batched float32
 * Householder QR on NVIDIA B200 (sm_100a) behind the entry points a binding of
 * the reference library already resolves. Each declaration names the reference
 * declaration it stands in for (paths inside the reference project).
 *
 * Matrices are float32, row-major and contiguous: a batch is its matrices one
 * after another. The caller allocates every output. A NaN or an infinity in a
 * matrix gives NaN output for that matrix alone.
 *
 * Pointers. The reference takes host-addressable memory (unified memory on
 * Apple silicon). Here a, q and r are either all CUDA device pointers on one
 * GPU, or all host pointers:
 *   device pointers  the work is enqueued on the calling thread's stream (see
 *                    metal_linalg_set_stream; the default stream if none was
 *                    set) and the call returns without waiting, as any CUDA
 *                    library call does;
 *   host pointers    the matrices are staged to the calling thread's device
 *                    (metal_linalg_set_device; GPU 0 by default) in chunks,
 *                    factored there and copied back; the call returns when q
 *                    and r are written, as the reference's does.
 * There is no CPU path in this build: nothing is ever computed on the host.
 */
#ifndef METAL_LINALG_C_API_H
#define METAL_LINALG_C_API_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* include/metal_linalg/c_api.h:19-24 */
typedef enum metal_linalg_status {
    METAL_LINALG_OK               = 0,
    METAL_LINALG_INVALID_ARGUMENT = 1,  /* a null pointer, pointers in different memories, a bad mode */
    METAL_LINALG_RUNTIME_ERROR    = 2,  /* a CUDA failure, or a kernel that gave up on a bounded wait */
    METAL_LINALG_OUT_OF_MEMORY    = 3
} metal_linalg_status;

/* include/metal_linalg/c_api.h:26-28. The message of the most recent failure on
 * this thread, or "" if there has been none. Valid until the next failure on
 * this thread. */
const char* metal_linalg_last_error(void);

/* ---------------------------------------------------------------------------
 * QR
 * ------------------------------------------------------------------------- */

/* include/metal_linalg/c_api.h:34-37. A = Q R with K = min(rows, cols):
 * q [batch, rows, K] with orthonormal columns, r [batch, K, cols] upper
 * triangular (every entry below the diagonal exactly 0). */
metal_linalg_status metal_linalg_qr(const float* a, uint32_t batch, uint32_t rows, uint32_t cols,
                                    float* q, float* r);

/* include/metal_linalg/c_api.h:39-50. The same with a mode, as numpy.linalg.qr's
 * and torch.linalg.qr's: METAL_LINALG_QR_REDUCED as above; METAL_LINALG_QR_R,
 * R alone, r [batch, K, cols], q unused (NULL is fine) and Q never formed;
 * METAL_LINALG_QR_COMPLETE, q [batch, rows, rows] square, r [batch, rows, cols]
 * with zero rows below K. */
typedef enum metal_linalg_qr_mode {
    METAL_LINALG_QR_REDUCED  = 0,
    METAL_LINALG_QR_R        = 1,
    METAL_LINALG_QR_COMPLETE = 2,
} metal_linalg_qr_mode;
metal_linalg_status metal_linalg_qr_with_mode(const float* a, uint32_t batch, uint32_t rows, uint32_t cols,
                                              metal_linalg_qr_mode mode, float* q, float* r);

/* No counterpart in the reference. The QR for callers that must not allocate
 * device memory at call time, or trigger the device-wide stall of a cudaFree:
 * a request loop with a latency budget, or a process whose framework has
 * already taken the GPU's memory for its own pool so that a library's
 * cudaMalloc may fail. metal_linalg_qr_with_mode keeps the scratch memory of
 * its block-per-matrix kernel in a workspace that grows on demand; this entry
 * point runs the same kernel on a scratch array built into the library image
 * instead (metal_linalg_qr_no_alloc_scratch_bytes() bytes, 32 MiB, held by every
 * GPU that loads the library until the process exits). It calls no cudaMalloc,
 * no cudaFree and no allocating library routine.
 *
 * a, q and r as metal_linalg_qr_with_mode's, but CUDA device pointers on one
 * GPU only; the work is enqueued on the calling thread's stream. Limits: at most
 * 1024 rows, and one matrix's scratch, 4 * (rows * cols + 1024 * ceil(min(rows,
 * cols) / 32)) bytes, must fit the array; beyond either the call fails with
 * METAL_LINALG_INVALID_ARGUMENT and a message that says which. Batches of any
 * size are fine: fewer matrices are in flight at once when the array holds
 * fewer slots.
 *
 * The first call on a GPU looks up the array's device address (once per GPU);
 * make that call before any stream capture. Every call on a GPU shares the one
 * array: each slot is rewritten in full before it is read, so nothing from an
 * earlier call leaks into a later one, but two calls that overlap on the GPU
 * (different streams or threads) race on it. Serialise them. */
metal_linalg_status metal_linalg_qr_no_alloc(const float* a, uint32_t batch, uint32_t rows, uint32_t cols,
                                             metal_linalg_qr_mode mode, float* q, float* r);
uint64_t            metal_linalg_qr_no_alloc_scratch_bytes(void);

/* ---------------------------------------------------------------------------
 * SVD: the QR's first caller inside the library
 * ------------------------------------------------------------------------- */

/* include/metal_linalg/c_api.h:59-63. Thin SVD A = U diag(s) Vt with K =
 * min(rows, cols): u [batch, rows, K], s [batch, K] descending, vt [batch, K,
 * cols]; u and vt both NULL for the singular values alone; info [batch] or
 * NULL. Pointers as for metal_linalg_qr: all on the host or all on one GPU.
 * Of the reference's SVD backends this library holds the QR-preconditioned
 * one alone (A = Q R by the QR above, then one-sided Jacobi on R), for K <= 128:
 * a larger K fails with METAL_LINALG_INVALID_ARGUMENT. */
metal_linalg_status metal_linalg_svd(const float* a, uint32_t batch, uint32_t rows, uint32_t cols,
                                     float* u, float* s, float* vt, uint32_t* info);

/* include/metal_linalg/c_api.h:96-102. An `info` word: bits 0-15 the sweeps
 * taken, bit 16 converged, bit 17 the matrix held a NaN or an infinity (its
 * outputs are all NaN), bit 18 rank-deficient. */
#define METAL_LINALG_INFO_SWEEPS(info)         ((info) & 0xFFFFu)
#define METAL_LINALG_INFO_CONVERGED(info)      (((info) >> 16) & 1u)
#define METAL_LINALG_INFO_NONFINITE(info)      (((info) >> 17) & 1u)
#define METAL_LINALG_INFO_RANK_DEFICIENT(info) (((info) >> 18) & 1u)

/* include/metal_linalg/c_api.h:175-176. "qr_jacobi", or "unavailable" for a
 * shape metal_linalg_svd refuses. The strings are static. */
const char* metal_linalg_svd_backend(uint32_t rows, uint32_t cols, uint32_t batch);
const char* metal_linalg_svdvals_backend(uint32_t rows, uint32_t cols, uint32_t batch);   /* values alone */

/* ---------------------------------------------------------------------------
 * The gated delta rule: a sequence of decayed reflections (no counterpart in
 * the reference)
 * ------------------------------------------------------------------------- */

/* Element types of the operators below. */
typedef enum metal_linalg_dtype {
    METAL_LINALG_FLOAT32     = 0,
    METAL_LINALG_BFLOAT16    = 1,
    METAL_LINALG_FLOAT16     = 2,
    METAL_LINALG_FLOAT8_E4M3 = 3,
    METAL_LINALG_FLOAT8_E5M2 = 4,
} metal_linalg_dtype;

/* The inputs of one call. For every value head h a state S [key_dim, value_dim]
 * (float32) runs through the tokens of its sequence,
 *
 *     S <- exp(g_t) S;   d_t = beta_t (v_t - S^T k_t);   S <- S + k_t d_t^T;   o_t = scale S^T q_t,
 *
 * that is S <- exp(g_t) (I - beta_t k_t k_t^T) S + beta_t k_t v_t^T: products of the
 * (generalised) reflections this library's QR is made of. Value head h reads q
 * and k of head h / (value_heads / heads).
 *
 * q, k [batch, tokens, heads, key_dim] and v [batch, tokens, value_heads,
 * value_dim] have element type `dtype` (float32, bfloat16 or float16), g and
 * beta [batch, tokens, value_heads] are float32. The last dimension of q, k and
 * v is contiguous; *_stride are the elements between batches, tokens and heads.
 * key_dim <= 128, value_dim <= 256, value_heads a multiple of heads and at most
 * 65535, tokens below 2^30, at most 65535 sequences (or batch rows).
 *
 * Sequences: with `sequences` 0 every batch row is one. Otherwise batch is 1 and
 * sequence i is the tokens cu_seqlens[i] .. cu_seqlens[i + 1] - 1 (index_bytes 4:
 * int32, 8: int64; sequences + 1 values, none falling). Tokens of no sequence,
 * before the first or behind the last one, give outputs and gradients of zero. A
 * sequence may be empty: its state passes through.
 *
 * All pointers are CUDA device pointers on one GPU: `device` names it, which the
 * caller vouches for, or is -1 and the call looks each pointer up (about 0.3 us a
 * pointer) and refuses those that are not. The work is enqueued on the
 * calling thread's stream (metal_linalg_set_stream). Nothing is allocated: the
 * caller gives the workspace, so that calls on several streams, or in several
 * captured graphs, each have their own. */
typedef struct metal_linalg_delta {
    uint32_t     batch, tokens, heads, value_heads, key_dim, value_dim;
    uint32_t     sequences;
    uint32_t     dtype;                                       /* a metal_linalg_dtype */
    uint32_t     index_bytes;                                 /* of cu_seqlens and slots: 4 or 8 */
    float        scale;
    int32_t      device;                                      /* the GPU that every pointer is on, vouched for by the caller; -1: look */
    uint32_t     reserved;                                    /* 0 */
    const void  *q, *k, *v;
    const float *g, *beta;
    const float *initial_state;                               /* [sequences or batch, value_heads, key_dim, value_dim], or NULL: zero */
    const void  *cu_seqlens;
    int64_t      q_stride[3], k_stride[3], v_stride[3], g_stride[3], beta_stride[3];
} metal_linalg_delta;

/* o [batch, tokens, value_heads, value_dim] of type `dtype` and final_state (as
 * initial_state; NULL if not wanted), both contiguous. workspace: at least
 * metal_linalg_gated_delta_rule_workspace_bytes(p, 0) bytes, on a 256-byte
 * boundary; the function returns 0 for a problem that the call would refuse. */
metal_linalg_status metal_linalg_gated_delta_rule(const metal_linalg_delta* p, void* o, float* final_state,
                                                  void* workspace, uint64_t workspace_bytes);
uint64_t            metal_linalg_gated_delta_rule_workspace_bytes(const metal_linalg_delta* p, int backward);

/* The gradients from d_o (type `dtype`, strides of batches, tokens and heads, last
 * dimension contiguous) and d_final_state (contiguous; NULL: zero). The forward is
 * computed again from the inputs, so nothing of it has to be kept. dq, dk, dv (type
 * `dtype`), dg, dbeta (float32) and d_initial_state (NULL if not wanted) are
 * contiguous in the shapes of what they belong to. */
metal_linalg_status metal_linalg_gated_delta_rule_backward(const metal_linalg_delta* p, const void* d_o,
                                                           const int64_t* d_o_stride, const float* d_final_state,
                                                           void* dq, void* dk, void* dv, float* dg, float* dbeta,
                                                           float* d_initial_state, void* workspace,
                                                           uint64_t workspace_bytes);

/* A few tokens a sequence, for decoding: batch row b runs its tokens through the
 * state in slot slots[b] of a pool [pool_size, value_heads, key_dim, value_dim]
 * (float32, pool_stride elements between slots, the rest contiguous), in place.
 * slots NULL: row b has slot b. A row whose slot is not in 0 .. pool_size - 1 is padding: its
 * outputs are zero and no state is touched. Rows that name the same slot are run
 * one after another in the order of the rows. initial_state, cu_seqlens and
 * sequences of `p` are not looked at. Needs no workspace. */
metal_linalg_status metal_linalg_gated_delta_step(const metal_linalg_delta* p, void* o, float* pool, int64_t pool_stride,
                                                  uint32_t pool_size, const void* slots);

/* ---------------------------------------------------------------------------
 * Products of matrices in 8-bit floating point with a scale for each block of
 * 128 (no counterpart in the reference)
 * ------------------------------------------------------------------------- */

/* x [batch, rows, cols] (float32, bfloat16 or float16; strides in elements between
 * matrices, rows and columns, one of the last two being 1) to `values` of type
 * `kind` (METAL_LINALG_FLOAT8_E4M3 or _E5M2; rows `values_stride` bytes apart,
 * matrices rows * values_stride) and a float32 scale for each block of
 * block_rows (1 or 128) x 128: scale = max(max|x| / M, 2^-126) with M the type's
 * largest value (448 or 57344), value = x / scale, a float32 rounded to the nearest, ties to even.
 * scales [batch, ceil(rows / block_rows), ceil(cols / 128)]. A block with a NaN or an
 * infinity stands for NaN throughout. (A transposed matrix is given by its strides.)
 * rows and cols are below 2^30, a matrix below 2^38 elements.
 * device: the GPU that every pointer is on, vouched for by the caller, or -1: the call
 * looks each pointer up (about 0.3 us a pointer) and refuses those that are not on one GPU. */
metal_linalg_status metal_linalg_quantize_fp8(const void* x, metal_linalg_dtype dtype, uint32_t batch, uint32_t rows,
                                              uint32_t cols, int64_t batch_stride, int64_t row_stride, int64_t col_stride,
                                              uint32_t block_rows, metal_linalg_dtype kind, void* values,
                                              uint64_t values_stride, float* scales, int device);

/* One operand of metal_linalg_matmul_fp8: `values` with k contiguous, rows
 * `stride` bytes and matrices `batch_stride` bytes apart (0: one matrix for the
 * whole batch; else a multiple of `stride`), all multiples of 16 as the address is; scales contiguous, one for each block of
 * block_rows (1 or 128) x 128, matrices ceil(rows / block_rows) * ceil(k / 128) floats apart (none
 * where batch_stride is 0). */
typedef struct metal_linalg_fp8_operand {
    const void*  values;
    const float* scales;
    uint64_t     stride, batch_stride;
    uint32_t     kind;                                        /* METAL_LINALG_FLOAT8_E4M3 or _E5M2 */
    uint32_t     block_rows;
} metal_linalg_fp8_operand;

/* c [batch, m, n] = a [batch, m, k] b [batch, n, k]^T (float32, bfloat16 or float16, contiguous):
 * products of 128 along k on the tensor cores, times both blocks' scales and summed in float32.
 * m, n and k are below 2^30, c below 2^28 tiles of 128 x 16 to 128 x 256.
 * device: as for metal_linalg_quantize_fp8. */
metal_linalg_status metal_linalg_matmul_fp8(const metal_linalg_fp8_operand* a, const metal_linalg_fp8_operand* b,
                                            uint32_t batch, uint32_t m, uint32_t n, uint32_t k, void* c,
                                            metal_linalg_dtype c_dtype, int device);

/* ---------------------------------------------------------------------------
 * CUDA placement (no counterpart in the reference, whose memory is unified)
 * ------------------------------------------------------------------------- */

/* The CUDA stream (a cudaStream_t as a pointer; NULL for the default stream)
 * this thread's calls on device pointers are enqueued on. Thread-local, and one
 * stream for every GPU: a stream belongs to the GPU it was created on, so set it
 * again before passing pointers that live on another GPU (a stream of the wrong
 * GPU makes the launch fail with METAL_LINALG_RUNTIME_ERROR). */
void  metal_linalg_set_stream(void* cuda_stream);
void* metal_linalg_stream(void);

/* The GPU this thread's calls on host pointers run on (device pointers run on
 * the GPU that owns them). Thread-local; 0 by default. Returns
 * METAL_LINALG_INVALID_ARGUMENT for an ordinal the machine does not have. */
metal_linalg_status metal_linalg_set_device(int device);
int                 metal_linalg_device(void);
int                 metal_linalg_device_count(void);

/* Waits for everything this thread has enqueued on its stream. Then reports, as
 * METAL_LINALG_RUNTIME_ERROR with the GPU, the kind of wait and the last shape
 * enqueued in the message, a kernel that gave up on one of its bounded waits on
 * any GPU this library has used since the last report. Such a kernel has
 * written NaN to the outputs of the matrices concerned, which by itself cannot
 * be told from a NaN in the input: this call (or the status of a host-pointer
 * call, which checks before it returns) is where the two differ. The
 * reference reports a failed GPU command the same way, with the shape
 * (src/qr_householder.mm:372-377, src/qr_blocked.mm:146-150, src/c_api.cpp:17-35). */
metal_linalg_status metal_linalg_synchronize(void);

/* No counterpart in the reference (whose buffers are the caller's). The library
 * keeps scratch memory per (GPU, stream) between calls, as large as the largest
 * call so far needed (hundreds of MB after a large blocked QR). This frees all
 * of it, after waiting for every GPU concerned, and stores the bytes freed in
 * *bytes_freed (may be NULL). Later calls allocate again. Call it after
 * destroying streams the library has seen, or to hand the memory back. Not to
 * be called while another thread is inside a call of this library. */
metal_linalg_status metal_linalg_release_workspaces(uint64_t* bytes_freed);

/* Testing aid, no counterpart in the reference: the next `count` matrices that
 * the grid-parallel blocked QR factors, or calls of metal_linalg_matmul_fp8, are
 * treated as if one of their tensor-core products had given up on a wait at once
 * (NaN outputs, the error at the next metal_linalg_synchronize). Nothing on the GPU is made to wait, fault or fail. */
void metal_linalg_inject_wait_failures(int count);

/* ---------------------------------------------------------------------------
 * Device and routing
 * ------------------------------------------------------------------------- */

/* include/metal_linalg/c_api.h:136-138,147. The device's name, e.g. "NVIDIA
 * B200" ("" if there is no GPU), and its multiprocessor count (0 if none). */
const char* metal_linalg_device_name(void);
uint32_t    metal_linalg_gpu_core_count(void);

/* include/metal_linalg/c_api.h:140-146. The reference prints a notice when its
 * routing table was not measured on the machine it runs on. This build has one
 * table, measured on B200; the notice is "" on a B200 and says so elsewhere. */
void        metal_linalg_set_calibration_notices(int enabled);
const char* metal_linalg_calibration_message(const char* decomposition);

/* include/metal_linalg/c_api.h:149-153. Kept for bindings that resolve them:
 * the host threads the staging of host-pointer calls may use. */
void     metal_linalg_set_cpu_threads(uint32_t n);
uint32_t metal_linalg_cpu_threads(void);

/* include/metal_linalg/c_api.h:155-161. The reference routes the calling
 * thread's calls to its CPU paths while this is non-zero. This build has no CPU
 * path: while it is non-zero, QR calls on this thread fail with
 * METAL_LINALG_RUNTIME_ERROR rather than run on the GPU behind the caller's back. */
void metal_linalg_set_cpu_only(int on);
int  metal_linalg_cpu_only(void);

/* include/metal_linalg/c_api.h:163-172. The backend a call of that shape uses
 * under the policy in effect: "unblocked" (a matrix to a warp or a thread
 * block) or "streaming_reduced" (a matrix spread over the grid: the blocked
 * compact-WY QR and the TSQR tree). Never "cpu". The strings are static. */
const char* metal_linalg_qr_backend(uint32_t rows, uint32_t cols, uint32_t batch);

/* The kernel behind that backend, by name: "small" (a matrix in a warp's
 * registers), "mid" (a matrix to a thread block), "tsqr" (a tall thin matrix as
 * a tree of row blocks), "blocked" (compact-WY panels and rank-k updates over
 * the grid). No counterpart in the reference. The strings are static. */
const char* metal_linalg_qr_kernel(uint32_t rows, uint32_t cols, uint32_t batch, metal_linalg_qr_mode mode);

/* include/metal_linalg/c_api.h:186-201. The routing policy, field for field as
 * the reference's so that a binding's struct keeps its layout. */
#define METAL_LINALG_NO_LIMIT 0xFFFFFFFFu

typedef struct metal_linalg_qr_policy {
    uint32_t m_crossover_small_batch;   /* k = min(rows, cols) from which a matrix is spread over */
    uint32_t m_crossover_large_batch;   /* the grid, for batches below / from batch_threshold */
    uint32_t batch_threshold;
    uint32_t gpu_max_k;                 /* the reference's GPU-or-CPU rule: kept, and read back, */
    uint32_t gpu_min_batch_times_k;     /* but without effect (every call runs on the GPU) */
    uint32_t gpu_min_batch;
    uint32_t gpu_cores;                 /* informational: multiprocessors */
    uint32_t concurrent_matrices;       /* informational: thread blocks of the mid kernel resident at once */
    uint32_t gpu_large_min_k;           /* a matrix is spread over the grid also from sqrt(rows k) >= this x sqrt(max(1, batch / 3)) */
    uint32_t gpu_large_max_batch;       /* (0: never) in a batch of at most this (0: any) */
    uint32_t gpu_min_k;                 /* without effect */
    uint32_t share_min_batch;           /* without effect (no CPU to share a batch with) */
} metal_linalg_qr_policy;

/* include/metal_linalg/c_api.h:301,308,319 */
metal_linalg_qr_policy metal_linalg_qr_policy_get(void);
void                   metal_linalg_qr_policy_set(const metal_linalg_qr_policy* p);
/* "tuned:<device>", "env:<variables>", "user" or "default:untuned-device (<device>)". */
const char*            metal_linalg_qr_policy_source(void);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* METAL_LINALG_C_API_H */
