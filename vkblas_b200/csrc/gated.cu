// gated.cu -- the gated feed-forward block and its backward pass.
//
//   g = X Wg^T, u = X Wu^T, h = act(g) * u            (X M x H, Wg and Wu F x H)
//   dG = dh * u * act'(g), dU = dh * act(g)
//   dx = dG Wg + dU Wu, dWg = dG^T X, dWu = dU^T X
//
// Sums and activations in fp32; dG and dU are rounded once to the operand type,
// which is what the products of the backward pass read.
#include "act.cuh"
#include "ops.cuh"
#include "simple.cuh"

namespace vkb {
namespace {

template <typename T>
struct Rows {                       // element (r, c) of a row-major matrix
    const T* p;
    uint32_t ld;
    __device__ float operator()(uint32_t r, uint32_t c) const {
        return Elem<T>::load(p + (size_t)r * ld + c);
    }
};
template <typename T>
struct Cols {                       // element (r, c) of its transpose
    const T* p;
    uint32_t ld;
    __device__ float operator()(uint32_t r, uint32_t c) const {
        return Elem<T>::load(p + (size_t)c * ld + r);
    }
    __device__ float operator()(int, uint32_t r, uint32_t c) const { return (*this)(r, c); }
};
template <typename T>
struct GateUp {
    Rows<T> w[2];
    __device__ float operator()(int i, uint32_t n, uint32_t k) const { return w[i](n, k); }
};
template <typename T, int ACT>
struct GatedOut {
    T *h, *g, *u;
    uint32_t ldh, ldg, ldu;
    __device__ void operator()(uint32_t m, uint32_t f, const float (&v)[2]) const {
        h[(size_t)m * ldh + f] = Elem<T>::from_f(act_fwd<ACT>(v[0]) * v[1]);
        if (g) g[(size_t)m * ldg + f] = Elem<T>::from_f(v[0]);
        if (u) u[(size_t)m * ldu + f] = Elem<T>::from_f(v[1]);
    }
};
template <typename T>
struct Store {
    T* c;
    uint32_t ldc;
    __device__ void operator()(uint32_t m, uint32_t n, const float (&v)[1]) const {
        c[(size_t)m * ldc + n] = Elem<T>::from_f(v[0]);
    }
};
// dx: k runs over dG's columns, then dU's.
template <typename T>
struct BothA {
    Rows<T> dg, du;
    uint32_t F;
    __device__ float operator()(uint32_t m, uint32_t k) const { return k < F ? dg(m, k) : du(m, k - F); }
};
template <typename T>
struct BothB {
    Cols<T> wg, wu;
    uint32_t F;
    __device__ float operator()(int, uint32_t n, uint32_t k) const {
        return k < F ? wg(n, k) : wu(n, k - F);
    }
};

struct GradArgs {
    const void *dh, *g, *u;
    uint32_t lddh, ldg, ldu;
    void *dg, *du;                  // M x F, row stride ldo (a multiple of 8)
    uint32_t ldo;
    uint32_t M, F;
};

// dG and dU from dh, g and u.  A pass over 5 M F elements, bound by memory:
// each thread takes 8 columns, with 128-bit accesses where VEC says that every
// row starts on 16 bytes.
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(256) gated_grad_kernel(const GradArgs a) {
    const uint32_t per = (a.F + 7) / 8;
    const uint64_t total = (uint64_t)a.M * per;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
        const uint32_t m = (uint32_t)(i / per), c = (uint32_t)(i - (uint64_t)m * per) * 8;
        const T* src[3] = {static_cast<const T*>(a.dh) + (size_t)m * a.lddh + c,
                           static_cast<const T*>(a.g) + (size_t)m * a.ldg + c,
                           static_cast<const T*>(a.u) + (size_t)m * a.ldu + c};
        const size_t o = (size_t)m * a.ldo + c;
        T in[3][8], dg[8], du[8];
        if (VEC && c + 8 <= a.F) {
#pragma unroll
            for (int j = 0; j < 3; j++)
                *reinterpret_cast<uint4*>(in[j]) = __ldcs(reinterpret_cast<const uint4*>(src[j]));
        } else {
#pragma unroll
            for (int j = 0; j < 3; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) in[j][e] = c + e < a.F ? src[j][e] : Elem<T>::from_f(0.f);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float act, d;
            act_both<ACT>(Elem<T>::to_f(in[1][e]), act, d);
            const float dh = Elem<T>::to_f(in[0][e]);
            dg[e] = Elem<T>::from_f(dh * Elem<T>::to_f(in[2][e]) * d);
            du[e] = Elem<T>::from_f(dh * act);
        }
        // ldo is F rounded up to 8: whole groups can be stored.
        *reinterpret_cast<uint4*>(static_cast<T*>(a.dg) + o) = *reinterpret_cast<const uint4*>(dg);
        *reinterpret_cast<uint4*>(static_cast<T*>(a.du) + o) = *reinterpret_cast<const uint4*>(du);
    }
}

template <typename F> cudaError_t by_act(int act, F&& f) {
    switch (act) {
        case VKBLAS_ACT_SILU: return f.template operator()<VKBLAS_ACT_SILU>();
        case VKBLAS_ACT_GELU: return f.template operator()<VKBLAS_ACT_GELU>();
        default: return f.template operator()<VKBLAS_ACT_GELU_TANH>();
    }
}

bool act_ok(int act) { return act >= VKBLAS_ACT_SILU && act <= VKBLAS_ACT_GELU_TANH; }

template <typename T> struct Forward {
    const vkblas_b200_gated_t& a;
    cudaStream_t s;
    template <int ACT> cudaError_t operator()() const {
        Rows<T> x{static_cast<const T*>(a.x), a.ldx};
        GateUp<T> w{{{static_cast<const T*>(a.w_gate), a.ldwg}, {static_cast<const T*>(a.w_up), a.ldwu}}};
        GatedOut<T, ACT> o{static_cast<T*>(a.h), static_cast<T*>(a.g), static_cast<T*>(a.u), a.ldh, a.ldg, a.ldu};
        return launch_simple<2>(a.M, a.F, a.H, x, w, o, s);
    }
};

struct BackPlan {
    void *dg, *du;
    uint32_t ldo;
    size_t bytes;
};
BackPlan back_plan(const vkblas_b200_gated_backward_t& a, void* ws) {
    Carver c(ws);
    BackPlan p;
    p.ldo = up8(a.F);
    p.dg = c.take<uint16_t>((size_t)a.M * p.ldo);
    p.du = c.take<uint16_t>((size_t)a.M * p.ldo);
    p.bytes = c.used;
    return p;
}

template <typename T> struct Grad {
    const GradArgs& g;
    bool vec;
    uint32_t blocks;
    cudaStream_t s;
    template <int ACT> cudaError_t operator()() const {
        if (vec) gated_grad_kernel<T, ACT, true><<<blocks, 256, 0, s>>>(g);
        else gated_grad_kernel<T, ACT, false><<<blocks, 256, 0, s>>>(g);
        count_launch();
        return cudaGetLastError();
    }
};

template <typename T>
cudaError_t backward(const vkblas_b200_gated_backward_t& a, const BackPlan& p, int num_sms, cudaStream_t s) {
    GradArgs ga{a.dh, a.g, a.u, a.lddh, a.ldg, a.ldu, p.dg, p.du, p.ldo, a.M, a.F};
    const bool vec = is_al(a.dh, 16) && is_al(a.g, 16) && is_al(a.u, 16) &&
                     (a.lddh | a.ldg | a.ldu) % 8 == 0;
    const uint64_t work = ((uint64_t)a.M * ((a.F + 7) / 8) + 255) / 256, cap = (uint64_t)num_sms * 16;
    cudaError_t e = by_act(a.act, Grad<T>{ga, vec, (uint32_t)(work < cap ? work : cap), s});
    const T *dg = static_cast<const T*>(p.dg), *du = static_cast<const T*>(p.du);
    if (e == cudaSuccess && a.dx) {
        BothA<T> A{{dg, p.ldo}, {du, p.ldo}, a.F};
        BothB<T> B{{static_cast<const T*>(a.w_gate), a.ldwg}, {static_cast<const T*>(a.w_up), a.ldwu}, a.F};
        e = launch_simple<1>(a.M, a.H, 2 * a.F, A, B, Store<T>{static_cast<T*>(a.dx), a.lddx}, s);
    }
    const Cols<T> X{static_cast<const T*>(a.x), a.ldx};
    if (e == cudaSuccess && a.dw_gate)
        e = launch_simple<1>(a.F, a.H, a.M, Cols<T>{dg, p.ldo}, X, Store<T>{static_cast<T*>(a.dw_gate), a.lddwg}, s);
    if (e == cudaSuccess && a.dw_up)
        e = launch_simple<1>(a.F, a.H, a.M, Cols<T>{du, p.ldo}, X, Store<T>{static_cast<T*>(a.dw_up), a.lddwu}, s);
    return e;
}

bool gated_ok(const vkblas_b200_gated_t* a) {
    return a && two_byte(a->dtype) && act_ok(a->act) && a->M && a->F && a->H &&
           mat_ok(a->x, a->ldx, a->H) && mat_ok(a->w_gate, a->ldwg, a->H) &&
           mat_ok(a->w_up, a->ldwu, a->H) && mat_ok(a->h, a->ldh, a->F) && !a->g == !a->u &&
           (!a->g || (mat_ok(a->g, a->ldg, a->F) && mat_ok(a->u, a->ldu, a->F)));
}

bool backward_ok(const vkblas_b200_gated_backward_t* a) {
    if (!a || !two_byte(a->dtype) || !act_ok(a->act) || !a->M || !a->F || !a->H) return false;
    if (!mat_ok(a->dh, a->lddh, a->F) || !mat_ok(a->g, a->ldg, a->F) || !mat_ok(a->u, a->ldu, a->F))
        return false;
    if (!a->dx && !a->dw_gate && !a->dw_up) return false;
    if (a->dx && (!mat_ok(a->dx, a->lddx, a->H) || !mat_ok(a->w_gate, a->ldwg, a->H) ||
                  !mat_ok(a->w_up, a->ldwu, a->H)))
        return false;
    if ((a->dw_gate || a->dw_up) && !mat_ok(a->x, a->ldx, a->H)) return false;
    return (!a->dw_gate || mat_ok(a->dw_gate, a->lddwg, a->H)) &&
           (!a->dw_up || mat_ok(a->dw_up, a->lddwu, a->H));
}

}  // namespace
}  // namespace vkb

using namespace vkb;
#define VKB_EXPORT extern "C" __attribute__((visibility("default")))

VKB_EXPORT size_t vkblas_b200_gated_workspace(const vkblas_b200_gated_t* a) { return 0; }

VKB_EXPORT vkblas_status_t vkblas_b200_gated(const vkblas_b200_gated_t* a, void* workspace,
                                             size_t workspace_bytes, void* stream) {
    if (!gated_ok(a)) return VKBLAS_ERR_PARAM;
    OpDevice d;
    if (!op_device(&d)) return VKBLAS_ERR_INIT;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return op_status(a->dtype == VKBLAS_DT_F16 ? by_act(a->act, Forward<__half>{*a, s})
                                               : by_act(a->act, Forward<__nv_bfloat16>{*a, s}));
}

VKB_EXPORT size_t vkblas_b200_gated_backward_workspace(const vkblas_b200_gated_backward_t* a) {
    return a && a->M && a->F ? back_plan(*a, nullptr).bytes : 0;
}

VKB_EXPORT vkblas_status_t vkblas_b200_gated_backward(const vkblas_b200_gated_backward_t* a,
                                                      void* workspace, size_t workspace_bytes,
                                                      void* stream) {
    if (!backward_ok(a)) return VKBLAS_ERR_PARAM;
    const BackPlan p = back_plan(*a, workspace);
    if (!ws_ok(workspace, workspace_bytes, p.bytes)) return VKBLAS_ERR_PARAM;
    OpDevice d;
    if (!op_device(&d)) return VKBLAS_ERR_INIT;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return op_status(a->dtype == VKBLAS_DT_F16 ? backward<__half>(*a, p, d.num_sms, s)
                                               : backward<__nv_bfloat16>(*a, p, d.num_sms, s));
}
