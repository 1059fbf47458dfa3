// ops.cuh -- what the fused language-model products (gated.cu, xent.cu, q4.cu)
// share: argument checks, the device record, the workspace carver.
#pragma once
#include "common.cuh"
#include "vkblas_b200.h"

namespace vkb {

// The current device's record for an operator: SM count and status word.
// False without an sm_100 device.  The first use on a device allocates the
// status word; that is allowed during stream capture, too.
struct OpDevice {
    int num_sms;
    int* status;
};
bool op_device(OpDevice* d);
// SM count of the current device, 148 when there is none (workspace sizes are
// then the ones a B200 needs).
int op_num_sms();

inline bool two_byte(int dtype) { return dtype == VKBLAS_DT_F16 || dtype == VKBLAS_DT_BF16; }
inline bool is_al(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
// A 2-byte operand of `cols`-long rows: present, element-aligned, rows apart.
inline bool mat_ok(const void* p, uint32_t ld, uint32_t cols) { return p && is_al(p, 2) && ld >= cols; }
// Sizes that the kernels' 32-bit signed tile coordinates reach, with a tile to spare.
inline bool size_ok(uint32_t n) { return n > 0 && n < 0x7FFFFE00u; }
inline size_t up256(size_t b) { return (b + 255) / 256 * 256; }
inline uint32_t up8(uint32_t v) { return (v + 7u) & ~7u; }
inline vkblas_status_t op_status(cudaError_t e) {
    if (e == cudaSuccess) return VKBLAS_OK;
    cudaGetLastError();
    return e == cudaErrorInvalidValue || e == cudaErrorInvalidConfiguration ? VKBLAS_ERR_PARAM
                                                                            : VKBLAS_ERR_INIT;
}

// Launches a kernel that waits in griddepcontrol.wait before its first global access as
// the programmatic dependent of the kernel ahead on the stream, so that its launch and
// set-up overlap that kernel's end.
template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kern)(P...), uint32_t grid, uint32_t block, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(grid);
    c.blockDim = dim3(block);
    c.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = at;
    c.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&c, kern, args...);
    count_launch();
    return e;
}

// Loads for kernels launched by launch_pdl.  Such a kernel is resident while kernels before
// it still write what it reads after its wait, so that memory is not read-only for the
// kernel's lifetime, as the .nc path (__ldg) wants it: lines an SM's L1 holds of it may be
// old, and the compiler may move such a load ahead of the wait.  These are ordinary loads
// that stay behind it.  What no such kernel writes may use the .nc path.
__device__ __forceinline__ uint4 ld16(const void* p) { return *static_cast<const uint4*>(p); }
// 16 bytes that are read once: past L1, in 256-byte L2 fetches.
__device__ __forceinline__ uint4 ld16_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// Eight 2-byte elements at any alignment, zeros after the first `left`.
__device__ __forceinline__ uint4 gather8(const uint16_t* p, int64_t left) {
    uint32_t e[8];
#pragma unroll
    for (int i = 0; i < 8; i++) e[i] = i < left ? (uint32_t)p[i] : 0u;
    return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
}

// Hands out 256-byte aligned pieces of the caller's workspace; with a null
// base it only counts, which is how the _workspace functions size it.
struct Carver {
    char* base;
    size_t used = 0;
    explicit Carver(void* p) : base(static_cast<char*>(p)) {}
    template <typename T> T* take(size_t n) {
        T* r = reinterpret_cast<T*>(base ? base + used : nullptr);
        used += up256(n * sizeof(T));
        return r;
    }
};
// Whether a workspace holds what a plan took.
inline bool ws_ok(const void* p, size_t bytes, size_t need) {
    return need == 0 || (p && is_al(p, 256) && bytes >= need);
}

// One tensor-core GEMM of the engine, C = alpha op(A) op(B) of 2-byte types, whose
// operands TMA can read, and its launch with room for the K split of its last wave
// (umma_split_workspace_bytes; null: no split).
inline GemmProblem product(int dtype, int op_a, int op_b, uint32_t M, uint32_t N, uint32_t K, const void* A,
                           uint32_t lda, const void* B, uint32_t ldb, void* C, uint32_t ldc) {
    GemmProblem p;
    p.dtype = dtype, p.op_a = op_a, p.op_b = op_b, p.M = M, p.N = N, p.K = K;
    p.alpha = 1.f, p.beta = 0.f, p.d_alpha = nullptr, p.d_beta = nullptr;
    p.A = A, p.lda = lda, p.B = B, p.ldb = ldb, p.C = C, p.ldc = ldc;
    p.batch = 1, p.sa = p.sb = p.sc = 0;
    return p;
}
inline cudaError_t launch_product(const GemmProblem& p, void* split, const OpDevice& d, cudaStream_t s) {
    return launch_umma_gemm(p, d.num_sms, d.status, nullptr, split, false, s);
}

}  // namespace vkb
