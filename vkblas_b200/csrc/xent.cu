// xent.cu -- softmax cross entropy of a linear head, forward and backward,
// without keeping the logits.
//
//   z = X W^T (X T x H, W V x H), lse_i = log sum_j exp z_ij, loss_i = lse_i - z_i,t
//   D = diag(dloss) (exp(z - lse) - onehot(t)), dx = D W, dW = D^T X
#include "ops.cuh"
#include "simple.cuh"

namespace vkb {
namespace {

constexpr uint32_t PIECE = 4096;     // vocabulary rows at a time

template <typename T>
struct Rows {
    const T* p;
    uint32_t ld;
    __device__ float operator()(uint32_t r, uint32_t c) const { return Elem<T>::load(p + (size_t)r * ld + c); }
    __device__ float operator()(int, uint32_t r, uint32_t c) const { return (*this)(r, c); }
};
template <typename T>
struct Cols {
    const T* p;
    uint32_t ld;
    __device__ float operator()(uint32_t r, uint32_t c) const { return Elem<T>::load(p + (size_t)c * ld + r); }
    __device__ float operator()(int, uint32_t r, uint32_t c) const { return (*this)(r, c); }
};
struct StoreF {
    float* z;
    uint32_t ld;
    __device__ void operator()(uint32_t m, uint32_t n, const float (&v)[1]) const { z[(size_t)m * ld + n] = v[0]; }
};
struct AddF {
    float* z;
    uint32_t ld;
    __device__ void operator()(uint32_t m, uint32_t n, const float (&v)[1]) const { z[(size_t)m * ld + n] += v[0]; }
};
template <typename T>
struct StoreScaled {
    T* c;
    uint32_t ldc;
    const float* scale;      // [1]: 1 / S
    __device__ void operator()(uint32_t m, uint32_t n, const float (&v)[1]) const {
        c[(size_t)m * ldc + n] = Elem<T>::from_f(v[0] * scale[1]);
    }
};

// Running maximum, sum and target logit of each row over the pieces.
struct Stat {
    float m, s, zt;
};
__global__ void row_stats(const float* z, uint32_t cols, uint32_t first, const int64_t* t, Stat* st, bool start) {
    const uint32_t row = blockIdx.x;
    __shared__ float sm[32], ss[32];
    float m = -INFINITY;
    for (uint32_t j = threadIdx.x; j < cols; j += blockDim.x) m = fmaxf(m, z[(size_t)row * PIECE + j]);
    const float mu = isinf(m) ? 0.f : m;
    float s = 0.f;
    for (uint32_t j = threadIdx.x; j < cols; j += blockDim.x) s += expf(z[(size_t)row * PIECE + j] - mu);
    for (int o = 16; o; o >>= 1) {
        const float m2 = __shfl_xor_sync(~0u, m, o), s2 = __shfl_xor_sync(~0u, s, o);
        const float M = fmaxf(m, m2), U = isinf(M) ? 0.f : M;
        s = s * expf((isinf(m) ? (m < 0 ? -INFINITY : 0.f) : m) - U) + s2 * expf((isinf(m2) ? (m2 < 0 ? -INFINITY : 0.f) : m2) - U);
        m = M;
    }
    if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = m, ss[threadIdx.x / 32] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        Stat r = start ? Stat{-INFINITY, 0.f, NAN} : st[row];
        for (uint32_t w = 0; w < blockDim.x / 32; w++) {
            const float M = fmaxf(r.m, sm[w]), U = isinf(M) ? 0.f : M;
            r.s = (r.s == 0.f ? 0.f : r.s * expf(r.m - U)) + (ss[w] == 0.f ? 0.f : ss[w] * expf(sm[w] - U));
            r.m = M;
        }
        const int64_t j = t[row] - first;
        if (j >= 0 && j < cols) r.zt = z[(size_t)row * PIECE + j];
        st[row] = r;
    }
}
__global__ void finish(const Stat* st, uint32_t T, const int64_t* t, int64_t ignore, float* loss, float* lse) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= T) return;
    const float l = (isinf(st[i].m) ? 0.f : st[i].m) + logf(st[i].s);
    if (lse) lse[i] = l;
    loss[i] = t[i] == ignore ? 0.f : l - st[i].zt;
}

// out[0] = S, out[1] = 1 / S: the power of two that brings the largest |dloss|
// of a kept row into [2^14, 2^15).
__global__ void grad_scale(const float* dloss, const int64_t* t, int64_t ignore, uint32_t T, float* out) {
    __shared__ float sm[32];
    float m = 0.f;
    for (uint32_t i = threadIdx.x; i < T; i += blockDim.x)
        if (t[i] != ignore && isfinite(dloss[i])) m = fmaxf(m, fabsf(dloss[i]));
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 0; w < blockDim.x / 32; w++) m = fmaxf(m, sm[w]);
        const int e = m > 0.f ? max(ilogbf(m), -100) : 14;
        out[0] = scalbnf(1.f, 14 - e);
        out[1] = scalbnf(1.f, e - 14);
    }
}
template <typename T>
__global__ void dlogits(const float* z, uint32_t rows, uint32_t cols, uint32_t first, const int64_t* t, int64_t ignore,
                        int64_t V, const float* dloss, const float* lse, const float* scale, T* d) {
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t r = (uint32_t)(i / cols), c = (uint32_t)(i % cols);
    if (r >= rows) return;
    float v = 0.f;
    if (t[r] != ignore) {
        const float k = t[r] < 0 || t[r] >= V ? NAN : dloss[r] * scale[0];
        v = k * (expf(z[(size_t)r * PIECE + c] - lse[r]) - (t[r] == (int64_t)first + c ? 1.f : 0.f));
    }
    d[(size_t)r * PIECE + c] = Elem<T>::from_f(v);
}
template <typename T>
__global__ void store_dx(const float* acc, uint32_t rows, uint32_t H, const float* scale, T* dx, uint32_t ld) {
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < (uint64_t)rows * H) dx[i / H * ld + i % H] = Elem<T>::from_f(acc[i] * scale[1]);
}

// X with the ignored rows cleared, in rows of ld (a multiple of 8): whatever a
// padding token's row holds, D^T X does not see it.
template <typename T>
__global__ void __launch_bounds__(256) kept_rows(const T* x, uint32_t ldx, uint32_t rows, uint32_t H,
                                                 const int64_t* t, int64_t ignore, T* out, uint32_t ld) {
    const uint64_t total = (uint64_t)rows * ld;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
        const uint32_t r = (uint32_t)(i / ld), c = (uint32_t)(i % ld);
        out[i] = c < H && t[r] != ignore ? x[(size_t)r * ldx + c] : Elem<T>::from_f(0.f);
    }
}

bool xent_ok(const vkblas_b200_linear_xent_t* a) {
    return a && two_byte(a->dtype) && a->T && a->V && a->H && mat_ok(a->x, a->ldx, a->H) &&
           mat_ok(a->w, a->ldw, a->H) && a->targets && is_al(a->targets, 8) && a->loss &&
           is_al(a->loss, 4) && is_al(a->lse, 4);
}
bool backward_ok(const vkblas_b200_linear_xent_backward_t* a) {
    return a && two_byte(a->dtype) && a->T && a->V && a->H && mat_ok(a->x, a->ldx, a->H) &&
           mat_ok(a->w, a->ldw, a->H) && a->targets && is_al(a->targets, 8) && a->dloss &&
           is_al(a->dloss, 4) && a->lse && is_al(a->lse, 4) && (a->dx || a->dw) &&
           (!a->dx || mat_ok(a->dx, a->lddx, a->H)) && (!a->dw || mat_ok(a->dw, a->lddw, a->H));
}

struct FwdPlan {
    float* z;
    Stat* st;
    size_t bytes;
};
FwdPlan fwd_plan(uint32_t T, void* ws) {
    Carver c(ws);
    FwdPlan p;
    p.z = c.take<float>((size_t)T * PIECE);
    p.st = c.take<Stat>(T);
    p.bytes = c.used;
    return p;
}
struct BwdPlan {
    float *z, *acc, *scale;
    void *d, *xk;
    uint32_t ldk;
    size_t bytes;
};
BwdPlan bwd_plan(const vkblas_b200_linear_xent_backward_t& a, void* ws) {
    Carver c(ws);
    BwdPlan p;
    p.z = c.take<float>((size_t)a.T * PIECE);
    p.d = c.take<uint16_t>((size_t)a.T * PIECE);
    p.acc = c.take<float>(a.dx ? (size_t)a.T * a.H : 0);
    p.scale = c.take<float>(2);
    p.ldk = up8(a.H);
    p.xk = c.take<uint16_t>(a.dw ? (size_t)a.T * p.ldk : 0);
    p.bytes = c.used;
    return p;
}

template <typename T>
cudaError_t forward(const vkblas_b200_linear_xent_t& a, const FwdPlan& p, cudaStream_t s) {
    const Rows<T> X{static_cast<const T*>(a.x), a.ldx};
    for (uint64_t f = 0; f < a.V; f += PIECE) {
        const uint32_t n = (uint32_t)(a.V - f < PIECE ? a.V - f : PIECE);
        const Rows<T> W{static_cast<const T*>(a.w) + f * a.ldw, a.ldw};
        cudaError_t e = launch_simple<1>(a.T, n, a.H, X, W, StoreF{p.z, PIECE}, s);
        if (e != cudaSuccess) return e;
        row_stats<<<a.T, 256, 0, s>>>(p.z, n, (uint32_t)f, a.targets, p.st, f == 0);
        count_launch();
    }
    finish<<<(a.T - 1) / 256 + 1, 256, 0, s>>>(p.st, a.T, a.targets, a.ignore_index, a.loss, a.lse);
    count_launch();
    return cudaGetLastError();
}

template <typename T>
cudaError_t backward(const vkblas_b200_linear_xent_backward_t& a, const BwdPlan& p, cudaStream_t s) {
    const Rows<T> X{static_cast<const T*>(a.x), a.ldx};
    T* d = static_cast<T*>(p.d);
    grad_scale<<<1, 1024, 0, s>>>(a.dloss, a.targets, a.ignore_index, a.T, p.scale);
    count_launch();
    if (a.dx) {
        cudaError_t e = cudaMemsetAsync(p.acc, 0, (size_t)a.T * a.H * 4, s);
        if (e != cudaSuccess) return e;
    }
    T* xk = static_cast<T*>(p.xk);
    if (a.dw) {
        kept_rows<T><<<1184, 256, 0, s>>>(X.p, a.ldx, a.T, a.H, a.targets, a.ignore_index, xk, p.ldk);
        count_launch();
    }
    for (uint64_t f = 0; f < a.V; f += PIECE) {
        const uint32_t n = (uint32_t)(a.V - f < PIECE ? a.V - f : PIECE);
        const T* w = static_cast<const T*>(a.w) + f * a.ldw;
        cudaError_t e = launch_simple<1>(a.T, n, a.H, X, Rows<T>{w, a.ldw}, StoreF{p.z, PIECE}, s);
        if (e != cudaSuccess) return e;
        dlogits<T><<<(uint32_t)(((uint64_t)a.T * n - 1) / 256 + 1), 256, 0, s>>>(
            p.z, a.T, n, (uint32_t)f, a.targets, a.ignore_index, a.V, a.dloss, a.lse, p.scale, d);
        count_launch();
        if (a.dx) e = launch_simple<1>(a.T, a.H, n, Rows<T>{d, PIECE}, Cols<T>{w, a.ldw}, AddF{p.acc, a.H}, s);
        if (e == cudaSuccess && a.dw)
            e = launch_simple<1>(n, a.H, a.T, Cols<T>{d, PIECE}, Cols<T>{xk, p.ldk},
                                 StoreScaled<T>{static_cast<T*>(a.dw) + f * a.lddw, a.lddw, p.scale}, s);
        if (e != cudaSuccess) return e;
    }
    if (a.dx) {
        store_dx<T><<<(uint32_t)(((uint64_t)a.T * a.H - 1) / 256 + 1), 256, 0, s>>>(
            p.acc, a.T, a.H, p.scale, static_cast<T*>(a.dx), a.lddx);
        count_launch();
    }
    return cudaGetLastError();
}

}  // namespace
}  // namespace vkb

using namespace vkb;
#define VKB_EXPORT extern "C" __attribute__((visibility("default")))

VKB_EXPORT size_t vkblas_b200_linear_xent_workspace(const vkblas_b200_linear_xent_t* a) {
    return a ? fwd_plan(a->T, nullptr).bytes : 0;
}

VKB_EXPORT vkblas_status_t vkblas_b200_linear_xent(const vkblas_b200_linear_xent_t* a, void* workspace,
                                                   size_t workspace_bytes, void* stream) {
    if (!xent_ok(a)) return VKBLAS_ERR_PARAM;
    const FwdPlan p = fwd_plan(a->T, workspace);
    if (!ws_ok(workspace, workspace_bytes, p.bytes)) return VKBLAS_ERR_PARAM;
    OpDevice d;
    if (!op_device(&d)) return VKBLAS_ERR_INIT;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return op_status(a->dtype == VKBLAS_DT_F16 ? forward<__half>(*a, p, s) : forward<__nv_bfloat16>(*a, p, s));
}

VKB_EXPORT size_t vkblas_b200_linear_xent_backward_workspace(const vkblas_b200_linear_xent_backward_t* a) {
    return a ? bwd_plan(*a, nullptr).bytes : 0;
}

VKB_EXPORT vkblas_status_t vkblas_b200_linear_xent_backward(const vkblas_b200_linear_xent_backward_t* a,
                                                            void* workspace, size_t workspace_bytes,
                                                            void* stream) {
    if (!backward_ok(a)) return VKBLAS_ERR_PARAM;
    const BwdPlan p = bwd_plan(*a, workspace);
    if (!ws_ok(workspace, workspace_bytes, p.bytes)) return VKBLAS_ERR_PARAM;
    OpDevice d;
    if (!op_device(&d)) return VKBLAS_ERR_INIT;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return op_status(a->dtype == VKBLAS_DT_F16 ? backward<__half>(*a, p, s) : backward<__nv_bfloat16>(*a, p, s));
}
