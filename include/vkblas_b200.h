/* vkblas_b200.h -- B200-specific extensions of the vkblas C API.
 *
 * These entry points have no counterpart in the reference's vkblas.h (its
 * engine was synchronous, single-stream and single-device).  They expose what
 * a stream-ordered CUDA library needs: a stream per calling thread, device
 * resident alpha/beta, kernel-path control for tests and benchmarks, the
 * device status word of the bounded waits, and the multi-GPU shard planner.
 */
#pragma once
#include "vkblas.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum { VKBLAS_DT_F32 = 0, VKBLAS_DT_F16 = 1, VKBLAS_DT_BF16 = 2 } vkblas_dtype_t;

/* Kernel families.  AUTO lets the dispatcher choose. */
typedef enum {
    VKBLAS_PATH_AUTO = 0,
    VKBLAS_PATH_SIMT = 1,   /* exact SIMT GEMM: sequential fp32 fmaf per output      */
    VKBLAS_PATH_TC = 2,     /* tcgen05 GEMM: kind::f16 (fp16/bf16) or 3xTF32 (fp32)   */
    VKBLAS_PATH_GEMV = 3    /* split-K decode GEMV (M <= 16, op_b == T, 2-byte types) */
} vkblas_path_t;

/* Generic entry used by the hipBLAS shim.  alpha and beta point to fp32
 * scalars in host memory (scalars_on_device == 0) or device memory (1); in
 * the device case the kernels read them, nothing is copied to the host.
 * stream: a cudaStream_t (NULL = legacy default stream). */
vkblas_status_t vkblas_gemm_ex(vkblas_dtype_t dtype, vkblas_op_t op_a, vkblas_op_t op_b,
                               uint32_t M, uint32_t N, uint32_t K,
                               const float* alpha, const float* beta, int scalars_on_device,
                               const void* A, uint32_t lda, const void* B, uint32_t ldb,
                               void* C, uint32_t ldc, uint32_t batch,
                               int64_t stride_a, int64_t stride_b, int64_t stride_c,
                               void* stream);

/* Frees this library's scratch workspaces on the current device: the ones
 * bound to `stream` (a cudaStream_t; NULL = legacy default stream) when
 * all == 0, or every stream's when all != 0.  Workspaces are grow-only and
 * kept per (device, stream) -- the 3xTF32 operand planes of a 4096^3 SGEMM
 * take 256 MB -- so a caller that ran GEMMs on many streams, or on a stream it
 * has destroyed, calls this to give the memory back; the next call that needs
 * scratch allocates it again.  Synchronises the device first.  Must not run
 * while another thread issues calls on this device.  Returns 0, or -1 when
 * no CUDA device state is available.  No counterpart in the reference. */
int vkblas_b200_release_workspaces(void* stream, int all);

/* Split-K decode GEMV that allocates nothing.  No counterpart in the
 * reference.  For callers that cannot let a library call cudaMalloc (work
 * inside a framework's allocator or memory pool, or decode loops where a
 * device-synchronising cudaFree/cudaMalloc of a growing workspace is not
 * acceptable).  Computes, for 2-byte dtype (VKBLAS_DT_F16 or VKBLAS_DT_BF16),
 *     C[m*ldc + n] = alpha * sum_k X[m*ldx + k] * W[n*ldw + k] + beta * C[m*ldc + n]
 * i.e. vkblas_gemm_f16/bf16(VKBLAS_OP_N, VKBLAS_OP_T, M, N, K, ...) with
 * batch 1, on `stream` (a cudaStream_t; NULL = legacy default stream), with
 * the K range split into `splitk` (1..16) segments.  Scratch is a fixed 4 MiB
 * array inside the library (held by every GPU that loads it until exit):
 * splitk*M*N*4 must fit in 4 MiB - 64 KiB and N in 16384*16 rows, and
 * M <= 16, K, ldx, ldw multiples of 8, X and W 16-byte aligned; otherwise
 * VKBLAS_ERR_PARAM and nothing is enqueued.  All calls on a device share the
 * array: calls whose kernels overlap on the GPU race (order them on one
 * stream).  The first call on a device looks the array up
 * (cudaGetSymbolAddress); make it before any stream capture. */
vkblas_status_t vkblas_gemv_splitk_noalloc(vkblas_dtype_t dtype, uint32_t M, uint32_t N,
                                           uint32_t K, float alpha, const void* X, uint32_t ldx,
                                           const void* W, uint32_t ldw, float beta, void* C,
                                           uint32_t ldc, uint32_t splitk, void* stream);

/* Replicated-output GEMM for data-parallel sharding.  No counterpart in the
 * reference (its engine drove one device).  Computes the engine call
 * (dtype, op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch,
 * stride_a/b/c) on the tcgen05 path, on `stream` (a cudaStream_t; NULL =
 * legacy default stream), and writes every element of C it produces also to
 * each of the `npeers` (0..7) buffers in peer_C, at the same element offset
 * from peer_C[j] as from C.  peer_C[j] are addresses valid in this process
 * (another GPU's memory mapped by CUDA IPC, over NVLink); the beta term reads
 * only C.  The peer stores are fenced system-wide before the kernels end;
 * the caller orders them before a peer reads its buffer with a collective
 * on `stream` after this call (a one-element NCCL all-reduce does).
 * VKBLAS_ERR_PARAM: unknown dtype, more than 7 peers, a null peer, or what
 * the engine rejects.  VKBLAS_ERR_FALLBACK (nothing launched, C and the
 * peers untouched): the problem cannot run on the tensor-core path (operand
 * alignment; a 2-byte problem with M <= 64 and N >= 128, which runs
 * transposed; scratch that cannot be had); the caller computes C and gathers
 * it another way. */
vkblas_status_t vkblas_b200_gemm_replicated(vkblas_dtype_t dtype, vkblas_op_t op_a,
                                            vkblas_op_t op_b, uint32_t M, uint32_t N, uint32_t K,
                                            float alpha, const void* A, uint32_t lda,
                                            const void* B, uint32_t ldb, float beta, void* C,
                                            uint32_t ldc, uint32_t batch, int64_t stride_a,
                                            int64_t stride_b, int64_t stride_c,
                                            void* const* peer_C, uint32_t npeers, void* stream);

/* ------------------------------------------------ fused language-model products
 *
 * Three products fused with what follows them in a language model.  No
 * counterpart in the reference.  All take 2-byte operands (VKBLAS_DT_F16 or
 * VKBLAS_DT_BF16; every operand of a call has that type unless stated),
 * row-major, with leading dimensions in elements; weights are stored as the
 * decode GEMV takes them, one row of K contiguous elements per output.  Sums,
 * softmax statistics and activations are held in fp32.  Any sizes (below 2^31 -
 * 512), leading dimensions (at least the row length) and element-aligned addresses
 * are taken; leading dimensions that are multiples of 8 and 16-byte aligned
 * addresses run fastest, other inputs are first copied into the workspace (the
 * one-token forms read them as they are).
 *
 * Calls enqueue on `stream` (a cudaStream_t; NULL = legacy default stream) on
 * the current device and neither allocate nor synchronise.  Scratch is the
 * caller's: `workspace` (256-byte aligned, at least the bytes that the
 * _workspace function gives for the same struct; NULL when that is 0) belongs
 * to the call until its work on the stream is done, so calls that may overlap,
 * and captured graphs that may run at the same time, need one each.  Outputs
 * must not overlap inputs, the workspace or each other.
 *
 * VKBLAS_ERR_PARAM: a size that is zero or too large, an unknown type or activation, a null or
 * misaligned pointer, a leading dimension below the row length, a workspace
 * that is too small.  VKBLAS_ERR_INIT: no sm_100 device, or a launch failed. */

typedef enum {
    VKBLAS_ACT_SILU = 0,         /* g / (1 + exp(-g))                                         */
    VKBLAS_ACT_GELU = 1,         /* g * (1 + erf(g / sqrt 2)) / 2                             */
    VKBLAS_ACT_GELU_TANH = 2     /* g * (1 + tanh(sqrt(2/pi) (g + 0.044715 g^3))) / 2         */
} vkblas_act_t;

/* Gated feed-forward block: with g = X Wg^T and u = X Wu^T,
 *     h[m, f] = act(g[m, f]) * u[m, f]
 * in one kernel.  X is M x H, Wg and Wu are F x H, h is M x F.  With `g` and
 * `u` given (both or neither), g and u are stored too, for the backward pass. */
typedef struct {
    vkblas_dtype_t dtype;
    vkblas_act_t act;
    uint32_t M, F, H;
    const void* x;      uint32_t ldx;
    const void* w_gate; uint32_t ldwg;
    const void* w_up;   uint32_t ldwu;
    void* h;            uint32_t ldh;
    void* g;            uint32_t ldg;    /* may be NULL, with u */
    void* u;            uint32_t ldu;
} vkblas_b200_gated_t;
size_t vkblas_b200_gated_workspace(const vkblas_b200_gated_t* a);
vkblas_status_t vkblas_b200_gated(const vkblas_b200_gated_t* a, void* workspace,
                                  size_t workspace_bytes, void* stream);

/* Its backward pass from the stored g and u and the gradient dh of h:
 *     dG = dh * u * act'(g),  dU = dh * act(g)   (rounded to the operand type, as the
 *         products read them; fp16 after a scaling by a power of two, which the products
 *         take back, that brings the largest finite value of both into [2^14, 2^15))
 *     dx = dG Wg + dU Wu,  dWg = dG^T X,  dWu = dU^T X
 * Any of dx, dw_gate, dw_up may be NULL and is then not computed (at least one
 * is given); w_gate and w_up are read for dx only, x for the weights only. */
typedef struct {
    vkblas_dtype_t dtype;
    vkblas_act_t act;
    uint32_t M, F, H;
    const void* dh;     uint32_t lddh;
    const void* g;      uint32_t ldg;
    const void* u;      uint32_t ldu;
    const void* x;      uint32_t ldx;
    const void* w_gate; uint32_t ldwg;
    const void* w_up;   uint32_t ldwu;
    void* dx;           uint32_t lddx;
    void* dw_gate;      uint32_t lddwg;
    void* dw_up;        uint32_t lddwu;
} vkblas_b200_gated_backward_t;
size_t vkblas_b200_gated_backward_workspace(const vkblas_b200_gated_backward_t* a);
vkblas_status_t vkblas_b200_gated_backward(const vkblas_b200_gated_backward_t* a, void* workspace,
                                           size_t workspace_bytes, void* stream);

/* Softmax cross entropy of a linear head, without keeping the logits:
 *     z = X W^T,  lse[i] = log sum_j exp z[i, j],  loss[i] = lse[i] - z[i, targets[i]]
 * X is T x H, W is V x H; loss and lse are T fp32 values.  A row whose target
 * is `ignore_index` has loss 0; one whose target is neither that nor in [0, V)
 * has loss NaN (its lse is still right).  lse may be NULL. */
typedef struct {
    vkblas_dtype_t dtype;
    uint32_t T, V, H;
    const void* x;          uint32_t ldx;
    const void* w;          uint32_t ldw;
    const int64_t* targets;
    int64_t ignore_index;
    float* loss;
    float* lse;
} vkblas_b200_linear_xent_t;
size_t vkblas_b200_linear_xent_workspace(const vkblas_b200_linear_xent_t* a);
vkblas_status_t vkblas_b200_linear_xent(const vkblas_b200_linear_xent_t* a, void* workspace,
                                        size_t workspace_bytes, void* stream);

/* Its backward pass from the forward pass's lse and the gradients dloss of the
 * T losses (fp32; for a mean over n rows, 1/n each):
 *     D = diag(dloss) (exp(z - lse) - onehot(targets)),  dx = D W,  dW = D^T X
 * The logits are computed again, as the forward pass sums them, in pieces of the vocabulary; D is
 * rounded to the operand type after a scaling by a power of two that keeps it in range.  Where
 * the target has nearly all the probability, what is left is as exact as lse (2^-24 of it).
 * Ignored rows give no gradient; a row with a target outside [0, V) gives NaN.
 * dx or dw may be NULL and is then not computed (one is given). */
typedef struct {
    vkblas_dtype_t dtype;
    uint32_t T, V, H;
    const float* dloss;
    const float* lse;
    const void* x;          uint32_t ldx;
    const void* w;          uint32_t ldw;
    const int64_t* targets;
    int64_t ignore_index;
    void* dx;               uint32_t lddx;
    void* dw;               uint32_t lddw;
} vkblas_b200_linear_xent_backward_t;
size_t vkblas_b200_linear_xent_backward_workspace(const vkblas_b200_linear_xent_backward_t* a);
vkblas_status_t vkblas_b200_linear_xent_backward(const vkblas_b200_linear_xent_backward_t* a,
                                                 void* workspace, size_t workspace_bytes,
                                                 void* stream);

/* 4-bit weights with group scales.  Weight (n, k) stands for
 *     scales[n, k / group] * (q[n, k] - zeros[n, k / group])
 * with q and zeros in 0..15 (zeros are 8 when there are none) and `group` a
 * multiple of 32.  vkblas_b200_q4_pack lays a matrix out once for the GEMV:
 * q is N rows of ldq bytes, two weights a byte, the even k in the low half;
 * scales (type `dtype`) and zeros (bytes; only the low 4 bits are read) are N x
 * ceil(K / group) with row strides lds and ldz in elements.  `packed` is the
 * caller's, 256-byte aligned, vkblas_b200_q4_bytes(w) bytes (0: bad sizes). */
typedef struct {
    vkblas_dtype_t dtype;        /* of scales and activations */
    uint32_t N, K, group;
    int has_zeros;
    const void* packed;          /* read by the products; not by q4_bytes and q4_pack */
} vkblas_b200_q4_t;
size_t vkblas_b200_q4_bytes(const vkblas_b200_q4_t* w);
vkblas_status_t vkblas_b200_q4_pack(const vkblas_b200_q4_t* w, const uint8_t* q, uint32_t ldq,
                                    const void* scales, uint32_t lds, const uint8_t* zeros,
                                    uint32_t ldz, void* packed, void* stream);
/* Y[m*ldy + n] = alpha * sum_k X[m*ldx + k] * weight(n, k) + beta * Y[m*ldy + n],
 * M <= 16 (else VKBLAS_ERR_PARAM); Y is not read when beta == 0.  No workspace. */
vkblas_status_t vkblas_b200_gemv_q4(const vkblas_b200_q4_t* w, uint32_t M, float alpha,
                                    const void* X, uint32_t ldx, float beta, void* Y, uint32_t ldy,
                                    void* stream);

/* Stream used by the vkblas_gemm_* calls made from the calling thread
 * (thread-local; default NULL = legacy default stream). */
void vkblas_set_stream(void* stream);
void* vkblas_get_stream(void);

/* Thread-local kernel-path override (VKBLAS_PATH_AUTO by default).  A forced
 * path that cannot run the call (alignment, shape) makes the call return
 * VKBLAS_ERR_FALLBACK instead of silently taking another path. */
void vkblas_b200_set_path(int path);
int vkblas_b200_get_path(void);
/* Path taken by the last successful call on this thread (vkblas_path_t). */
int vkblas_b200_last_path(void);
/* K-split count of that call: the GEMV split-K factor, or for the tensor-core
 * path the number of K ranges the tiles of its last, partial wave were cut
 * into (their partial sums are added by a second kernel); 1 = no split. */
int vkblas_b200_last_split(void);
/* 1 when that call ran on 2-CTA clusters (tcgen05 cta_group::2, 256-row
 * tiles: each CTA loads half of the B tile), else 0. */
int vkblas_b200_last_pair(void);
/* N width of that call's tensor-core tile: 256 for fp16/bf16 and for 3xTF32
 * on CTA pairs with N >= 256, 128 for other 3xTF32 tiles, 64 for small-M
 * transposed tiles (over the swapped problem); 0 when the call did not run on
 * the tensor-core path. */
int vkblas_b200_last_tile_n(void);
/* Thread-local split-K factor for the GEMV path: 0 = automatic, else 1..16. */
void vkblas_b200_set_splitk(int splitk);

/* Measurement hook (thread-local; NULL, NULL turns it off): while set, each
 * GEMM call made from this thread records the cudaEvent_t `start` on its
 * stream right before its main kernel (after the 3xTF32 split pre-pass, when
 * there is one) and `end` right after it (after the split-K reduce, when
 * there is one).  Timing those events gives the kernel's own duration inside
 * a stream of calls.  Both events must belong to the call's device. */
void vkblas_b200_set_kernel_events(void* start, void* end);

/* Device status word written by kernels whose bounded waits ran out (0 = no
 * error).  Synchronises the current device first.  clear != 0 resets it. */
int vkblas_b200_device_status(int clear);

/* Test hook for the bounded waits (thread-local, off by default): while on,
 * tcgen05 GEMMs launched from this thread leave their first shared-memory
 * stage unfilled and wait at most 20 ms, so the MMA warp's wait runs out, the
 * kernel records status 2 (MMA wait timeout) in the device status word and
 * every role unwinds; the context stays usable.  For tests only. */
void vkblas_b200_set_test_stall(int on);

/* Test hook for scratch-memory failure (thread-local, off by default): with
 * count > 0 the next `count` scratch requests made from this thread fail as a
 * failed cudaMalloc would, with count < 0 every request fails until the hook
 * is set to 0.  A call that then lacks its scratch runs without it where it
 * can (a GEMV or tensor-core GEMM without its K split; an fp32 GEMM on the
 * exact SIMT kernel instead of 3xTF32 when the path is automatic) or returns
 * VKBLAS_ERR_FALLBACK (path forced to VKBLAS_PATH_TC; the hipBLAS shim then
 * forwards the call).  For tests only. */
void vkblas_b200_set_test_alloc_fail(int count);

/* Number of kernels this library launched from the calling process (all
 * threads); used by tests and benchmarks to prove the native path ran. */
uint64_t vkblas_b200_launch_count(void);

/* Library version string. */
const char* vkblas_b200_version(void);

/* Tile and split plan of a tensor-core GEMM (pure host logic; no device is
 * touched).  For the engine call (dtype, op_a, op_b, M, N, K, batch) on a
 * device with `num_sms` SMs it reports the tiles the tcgen05 kernel would run
 * and how the tiles of the last, partial wave are cut along K.  allow_wide:
 * whether 256-wide 3xTF32 pair tiles may be chosen (the launch path allows
 * them when its kernel's register split fits and VKBLAS_TF32_WIDE is not 0).
 * The plan assumes the K-split is on (VKBLAS_TC_SPLIT) and its scratch can be
 * had.  Returns VKBLAS_ERR_PARAM for a zero size, num_sms < 1, an unknown dtype,
 * a null `out`, or 2^31 tiles or more (a call the tensor-core path rejects).
 * No counterpart in the reference. */
typedef struct {
    uint32_t tile_m;             /* rows of a tile: 128, or 256 on CTA pairs */
    uint32_t tile_n;             /* columns of a tile */
    uint32_t transposed;         /* 1: small-M 2-byte GEMM run as C^T = op(B)^T op(A)^T;
                                    tile_m, tile_n and tiles then refer to C^T */
    uint32_t pair;               /* 1: 2-CTA clusters (cta_group::2) */
    uint32_t tiles;              /* tiles over all batch entries */
    uint32_t full_tiles;         /* tiles computed whole (the full waves) */
    uint32_t splits;             /* K ranges each remaining tile is cut into; 1 = none */
    uint32_t kblocks;            /* k-blocks per tile: K / 32 (fp32) or K / 64, rounded up */
    uint32_t kblocks_per_split;  /* k-blocks per K range of a split tile */
    uint64_t partial_bytes;      /* fp32 partial-tile scratch of the split tiles */
    uint32_t tail_tiles;         /* tiles of the last wave run as two 256 x 128 halves each in a
                                    second, programmatically dependent grid (2-byte pair tiles
                                    whose last wave fills at most half the SM pairs); they
                                    follow the full_tiles whole tiles */
} vkblas_b200_tc_plan_t;
vkblas_status_t vkblas_b200_tc_plan(vkblas_dtype_t dtype, vkblas_op_t op_a, vkblas_op_t op_b,
                                    uint32_t M, uint32_t N, uint32_t K, uint32_t batch,
                                    int num_sms, int allow_wide, vkblas_b200_tc_plan_t* out);

/* Throughput microbenchmarks of the current device (no counterpart in the
 * reference's API; its test/fma_peak.c measured its FMA ceiling the same way).
 * Enqueues one launch of kernel `which` on `stream` (a cudaStream_t) that
 * runs `iters` rounds of only the instruction under test on every SM, and
 * stores the FLOP that launch performs in *flops; the caller times it with
 * CUDA events.  `status` is a device int that a bounded wait sets non-zero
 * if the tensor core's final commit never arrived.  VKBLAS_ERR_PARAM for an
 * unknown `which`, iters == 0 or null pointers; VKBLAS_ERR_INIT without an
 * sm_100 device. */
typedef enum {
    VKBLAS_PEAK_FFMA = 0,       /* fp32 fmaf, 2048 threads per SM                    */
    VKBLAS_PEAK_TF32 = 1,       /* tcgen05.mma kind::tf32, cta_group::1, 128x256x8   */
    VKBLAS_PEAK_TF32_PAIR = 2,  /* tcgen05.mma kind::tf32, cta_group::2, 256x256x8   */
    VKBLAS_PEAK_F16 = 3,        /* tcgen05.mma kind::f16,  cta_group::1, 128x256x16  */
    VKBLAS_PEAK_F16_PAIR = 4    /* tcgen05.mma kind::f16,  cta_group::2, 256x256x16  */
} vkblas_b200_peak_t;
vkblas_status_t vkblas_b200_peak_launch(int which, uint32_t iters, void* stream, int* status,
                                        double* flops);

/* Multi-GPU shard planner (pure host logic).  Splits `units` work units
 * (batch entries, or column blocks of `block` columns) into `world` contiguous
 * ranges as evenly as possible; returns this rank's [begin, begin+count).
 * Returns VKBLAS_ERR_PARAM for world < 1 or rank outside [0, world). */
vkblas_status_t vkblas_shard_range(uint64_t units, uint64_t block, int rank, int world,
                                   uint64_t* begin, uint64_t* count);

#ifdef __cplusplus
}
#endif
