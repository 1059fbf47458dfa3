// gated.cu -- the gated feed-forward block and its backward pass.
//
//   g = X Wg^T, u = X Wu^T, h = act(g) * u            (X M x H, Wg and Wu F x H)
//   dG = dh * u * act'(g), dU = dh * act(g)
//   dx = dG Wg + dU Wu, dWg = dG^T X, dWu = dU^T X
//
// Sums and activations in fp32; dG and dU are rounded once to the operand type,
// which is what the products of the backward pass read (fp16: after a scaling).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "act.cuh"
#include "umma_fused.cuh"

namespace vkb {
namespace {

// ------------------------------------------------------------- up to 16 tokens
// The decode form of the block, bound by the stream of both weight matrices
// (4 F H bytes).  It is the split-K GEMV of gemv.cu with one change: a warp's 16 MMA
// rows are 8 gate rows and the same 8 up rows, so that a lane ends up with
// both projections of its outputs and applies the activation in registers.  A
// CTA's KW warps split K and add their sums through shared memory in warp order.
struct TokenArgs {
    const void *x, *wg, *wu;
    uint32_t ldx, ldwg, ldwu;
    void *h, *g, *u;
    uint32_t ldh, ldg, ldu;
    uint32_t M, F, K;
};

template <typename T> __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight elements from p (k ones before the end of the row).  VEC: rows start on
// 16 bytes and K is a multiple of 8, so the eight are all there or none is.
template <bool VEC, bool STREAM>
__device__ __forceinline__ uint4 load8(const uint16_t* p, int64_t left, bool ok) {
    if (!ok || left <= 0) return make_uint4(0u, 0u, 0u, 0u);
    if constexpr (!VEC) return gather8(p, left);
    else if constexpr (STREAM) return ld16_stream(p);
    else return ld16(p);
}

template <typename T, int ACT, bool TWO, bool VEC, int KW>
__global__ void __launch_bounds__(KW * 32) gated_token_kernel(const TokenArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t f = blockIdx.x * 8 + g;
    const uint32_t per = ((a.K + KW - 1) / KW + 63) / 64 * 64;
    const uint32_t k0 = min(a.K, warp * per), k1 = min(a.K, k0 + per);
    const bool fok = f < a.F, x0ok = g < a.M, x1ok = TWO && g + 8 < a.M;
    const uint16_t* wg = static_cast<const uint16_t*>(a.wg) + (size_t)(fok ? f : 0) * a.ldwg;
    const uint16_t* wu = static_cast<const uint16_t*>(a.wu) + (size_t)(fok ? f : 0) * a.ldwu;
    const uint16_t* x0 = static_cast<const uint16_t*>(a.x) + (size_t)(x0ok ? g : 0) * a.ldx;
    const uint16_t* x1 = static_cast<const uint16_t*>(a.x) + (size_t)(x1ok ? g + 8 : 0) * a.ldx;
    float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
    // Two 64-wide chunks a step: eight 128-bit weight loads in flight a lane.  CTAs
    // start at different steps, so that they do not all read the same k offset of
    // their rows at a time (as in gemv.cu).
    const uint32_t nstep = (k1 - k0) / 128, rot = nstep ? blockIdx.x * 3u % nstep : 0u;
    auto chunk = [&](const uint4& lo, const uint4& hi, uint32_t k) {
        const uint32_t a0[4] = {lo.x, hi.x, lo.y, hi.y}, a1[4] = {lo.z, hi.z, lo.w, hi.w};
        const int64_t left = (int64_t)k1 - k;
        const uint4 xa = load8<VEC, false>(x0 + k, left, x0ok);
        mma16816<T>(d0, a0, xa.x, xa.y);
        mma16816<T>(d0, a1, xa.z, xa.w);
        if constexpr (TWO) {
            const uint4 xb = load8<VEC, false>(x1 + k, left, x1ok);
            mma16816<T>(d1, a0, xb.x, xb.y);
            mma16816<T>(d1, a1, xb.z, xb.w);
        }
    };
    for (uint32_t i = 0; i < nstep; i++) {
        const uint32_t ii = i + rot < nstep ? i + rot : i + rot - nstep;
        const uint32_t k = k0 + ii * 128 + 8 * t;
        uint4 w[4][2];
#pragma unroll
        for (uint32_t c = 0; c < 4; c++) {
            w[c][0] = load8<VEC, true>(wg + k + 32 * c, 8, fok);
            w[c][1] = load8<VEC, true>(wu + k + 32 * c, 8, fok);
        }
#pragma unroll
        for (uint32_t c = 0; c < 4; c++) chunk(w[c][0], w[c][1], k + 32 * c);
    }
    for (uint32_t kb = k0 + nstep * 128; kb < k1; kb += 32) {
        const uint32_t k = kb + 8 * t;
        const int64_t left = (int64_t)k1 - k;
        chunk(load8<VEC, true>(wg + k, left, fok), load8<VEC, true>(wu + k, left, fok), k);
    }
    __shared__ float red[KW][TWO ? 8 : 4][32];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        red[warp][i][lane] = d0[i];
        if (TWO) red[warp][4 + i][lane] = d1[i];
    }
    __syncthreads();
    // Warp 0 adds tokens 0-7, warp 1 tokens 8-15.  Of a lane's four sums the first two
    // are the gate of tokens 2t, 2t + 1, the others their up projection.
    if (warp >= (TWO ? 2u : 1u) || !fok) return;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[i] = red[0][warp * 4 + i][lane];
#pragma unroll
        for (int w = 1; w < KW; w++) v[i] = __fadd_rn(v[i], red[w][warp * 4 + i][lane]);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t m = warp * 8 + 2 * t + i;
        if (m >= a.M) continue;
        static_cast<T*>(a.h)[(size_t)m * a.ldh + f] = Elem<T>::from_f(act_fwd<ACT>(v[i]) * v[2 + i]);
        if (a.g) {
            static_cast<T*>(a.g)[(size_t)m * a.ldg + f] = Elem<T>::from_f(v[i]);
            static_cast<T*>(a.u)[(size_t)m * a.ldu + f] = Elem<T>::from_f(v[2 + i]);
        }
    }
}

// Up to 16 tokens (two MMA token tiles) run here, more on tcgen05.  Both at 4096 -> 14336: 1
// token 38.0 and 55.4 us, 16 tokens 41.7 and 43.4; 4096 -> 11008, 12 tokens, 31.9 and 52.1; 1024 ->
// 4096, 16 tokens, 4.7 and 10.7; 2048 -> 5461, 9 tokens, 11.0 and 24.4.
constexpr uint32_t TOKENS_MAX = 16;

// CTAs of a kernel that share an SM of the current device.
template <typename T, int ACT, bool TWO, bool VEC, int KW>
uint32_t resident() {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
    n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, gated_token_kernel<T, ACT, TWO, VEC, KW>, KW * 32, 0) !=
                cudaSuccess || n < 1)
            n = 1;
        known[dev].store(n, std::memory_order_relaxed);
    }
    return (uint32_t)n;
}

template <typename T> struct Token {
    const TokenArgs& a;
    bool vec;
    int num_sms;
    cudaStream_t s;
    // Warps a CTA: 4, 5, 6 or 8, whichever leaves the fewest CTA slots of an SM empty over
    // the waves of CTAs; the least where that is the same.  Measured (us, with 4 / 5 / 6 / 8):
    // 1 token 4096 -> 14336 39.7 / 38.0 / 39.3 / 42.2, 1024 -> 4096 4.8 / 4.7 / 4.3 / 3.8, 2048 ->
    // 8192 12.9 / 12.6 / 13.9 / 14.8; 4 tokens 4096 -> 11008 38.6 / 33.7 / 29.8 / 33.0; 9 tokens
    // 2048 -> 5461 11.9 / 10.8 / 11.0 / 14.0; 16 tokens 4096 -> 14336 46.6 / 41.7 / 46.1 / 46.8,
    // 1024 -> 4096 6.7 / 5.5 / 5.4 / 4.7; 12 tokens 4096 -> 11008 43.9 / 36.4 / 32.1 / 35.5.
    template <int ACT, bool TWO, bool VEC> cudaError_t go() const {
        const uint32_t ctas = (a.F - 1) / 8 + 1;
        const uint32_t on_sm[4] = {resident<T, ACT, TWO, VEC, 4>(), resident<T, ACT, TWO, VEC, 5>(),
                                   resident<T, ACT, TWO, VEC, 6>(), resident<T, ACT, TWO, VEC, 8>()};
        int best = 0;
        uint64_t taken = ~0ull;
        for (int i = 0; i < 4; i++) {
            const uint64_t slots = (uint64_t)on_sm[i] * (uint32_t)num_sms, all = ((ctas - 1) / slots + 1) * slots;
            if (all < taken) taken = all, best = i;
        }
        switch (best) {
            case 0: return launch_pdl(gated_token_kernel<T, ACT, TWO, VEC, 4>, ctas, 128, s, a);
            case 1: return launch_pdl(gated_token_kernel<T, ACT, TWO, VEC, 5>, ctas, 160, s, a);
            case 2: return launch_pdl(gated_token_kernel<T, ACT, TWO, VEC, 6>, ctas, 192, s, a);
            default: return launch_pdl(gated_token_kernel<T, ACT, TWO, VEC, 8>, ctas, 256, s, a);
        }
    }
    template <int ACT> cudaError_t operator()() const {
        if (vec) return a.M > 8 ? go<ACT, true, true>() : go<ACT, false, true>();
        return a.M > 8 ? go<ACT, true, false>() : go<ACT, false, false>();
    }
};

// ------------------------------------------------------------- more tokens
// Epilogue of the tcgen05 product (umma_fused.cuh): the first half of a tile's
// accumulator columns are gate projections, the second half the up projections of the
// same outputs.  The two warps of a lane quarter have 64 outputs each (32 of a tile of
// at most 64) and read 32 columns of each projection at a time; what they read past
// the tile is not stored.
template <typename T, int ACT, bool SAVE>
struct GatedEpi {
    static constexpr uint32_t SEG_KB = 0;
    static constexpr bool TWO_B = true;
    struct Args {
        fused::Out h, g, u;
    };
    template <typename A, typename R>
    static __device__ __forceinline__ void run(const fused::Params& p, const Args& a, const fused::Tile& t,
                                               A&& acquire, R&& release) {
        if (!acquire()) return;
        const uint32_t per = p.half > 64 ? 64 : 32, c0 = t.half * per;
        uint32_t h[32], gs[SAVE ? 32 : 1], us[SAVE ? 32 : 1];
#pragma unroll
        for (uint32_t c = 0; c < 2; c++) {
            if (c * 32 >= per || c0 + c * 32 >= p.half) break;
            uint32_t g[32], u[32];
            umma::tmem_ld_32x32b_x32(t.tmem + c0 + c * 32, g);
            umma::tmem_ld_32x32b_x32(t.tmem + p.half + c0 + c * 32, u);
            umma::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float g0 = __uint_as_float(g[2 * i]), g1 = __uint_as_float(g[2 * i + 1]);
                const float u0 = __uint_as_float(u[2 * i]), u1 = __uint_as_float(u[2 * i + 1]);
                h[c * 16 + i] = fused::pack2<T>(act_fwd<ACT>(g0) * u0, act_fwd<ACT>(g1) * u1);
                if constexpr (SAVE) {
                    gs[c * 16 + i] = fused::pack2<T>(g0, g1);
                    us[c * 16 + i] = fused::pack2<T>(u0, u1);
                }
            }
        }
        release();
        if (c0 >= p.half) return;
        const uint32_t n0 = t.nb * p.half + c0, width = min(per, p.half - c0);
        fused::store_rows(a.h, t, n0, width, h);
        if constexpr (SAVE) {
            fused::store_rows(a.g, t, n0, width, gs);
            fused::store_rows(a.u, t, n0, width, us);
        }
    }
};

struct GradArgs {
    const void *dh, *g, *u;
    uint32_t lddh, ldg, ldu;
    void *dg, *du;                  // M x F, row stride ldo (a multiple of 8)
    uint32_t ldo;
    uint32_t M, F;
    float* part;                    // fp16: the largest of |dG|, |dU| that each block of the first pass saw
    uint32_t parts;
    float* scale;                   // fp16: [0] = 1 / S, [1] = 0 (alpha and beta of the products)
};

// The largest value of a block of 256 threads, in all of them.
__device__ __forceinline__ float block_max(float m) {
    __shared__ float sm[8];
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = m;
    __syncthreads();
    for (int w = 0; w < 8; w++) m = fmaxf(m, sm[w]);
    return m;
}

// dG and dU from dh, g and u.  A pass over 5 M F elements, bound by memory (4096 x
// 14336, bf16: 97 us, 6.05 TB/s).  VEC, every row starts on 16 bytes: each thread takes 8
// neighbouring columns with 128-bit accesses.  Else a warp takes 256 columns, 32 at a
// time, so that its 2-byte accesses are neighbours.
//
// fp16 holds products of gradients and activations only after a scaling: dh * u passes 65504
// or vanishes below 6e-8 where dx and the weights' gradients, which the products bring back
// with x and W, are in range.  So dG and dU are stored times S, the power of two that brings the
// larger of their maxima into [2^14, 2^15), and the products divide by S in fp32.  MAX: the
// pass before, which finds the maxima (3 M F elements: with it the fp16 gradients at 4096 x 14336
// took 1573 us, bf16's 1461); non-finite values take no part.
template <typename T, int ACT, bool VEC, bool MAX>
__global__ void __launch_bounds__(256) gated_grad_kernel(const GradArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr bool SCALED = std::is_same<T, __half>::value;
    const T *dh = static_cast<const T*>(a.dh), *g = static_cast<const T*>(a.g), *u = static_cast<const T*>(a.u);
    T *dg = static_cast<T*>(a.dg), *du = static_cast<T*>(a.du);
    float most = 0.f, S = 1.f;
    if constexpr (SCALED && !MAX) {
        for (uint32_t i = threadIdx.x; i < a.parts; i += 256) most = fmaxf(most, a.part[i]);
        most = block_max(most);
        const int e = most > 0.f ? max(ilogbf(most), -100) : 14;
        S = scalbnf(1.f, 14 - e);
        if (blockIdx.x == 0 && threadIdx.x == 0) a.scale[0] = scalbnf(1.f, e - 14), a.scale[1] = 0.f;
    }
    auto one = [&](T dhv, T gv, T uv, T& dgv, T& duv) {
        float act, d;
        act_both<ACT>(Elem<T>::to_f(gv), act, d);
        const float x = Elem<T>::to_f(dhv), vg = x * Elem<T>::to_f(uv) * d, vu = x * act;
        if constexpr (MAX) {
            if (isfinite(vg)) most = fmaxf(most, fabsf(vg));
            if (isfinite(vu)) most = fmaxf(most, fabsf(vu));
        } else {
            dgv = Elem<T>::from_f(SCALED ? vg * S : vg);
            duv = Elem<T>::from_f(SCALED ? vu * S : vu);
        }
    };
    const uint32_t per = VEC ? (a.F + 7) / 8 : (a.F + 255) / 256 * 32;      // threads a row
    const uint64_t total = (uint64_t)a.M * per;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
        const uint32_t m = (uint32_t)(i / per), j = (uint32_t)(i - (uint64_t)m * per);
        const T *dhr = dh + (size_t)m * a.lddh, *gr = g + (size_t)m * a.ldg, *ur = u + (size_t)m * a.ldu;
        const size_t o = (size_t)m * a.ldo;
        if (VEC && j * 8 + 8 <= a.F) {
            T x[8], y[8], z[8], p[8], q[8];
            *reinterpret_cast<uint4*>(x) = __ldcs(reinterpret_cast<const uint4*>(dhr + j * 8));
            *reinterpret_cast<uint4*>(y) = __ldcs(reinterpret_cast<const uint4*>(gr + j * 8));
            *reinterpret_cast<uint4*>(z) = __ldcs(reinterpret_cast<const uint4*>(ur + j * 8));
#pragma unroll
            for (int e = 0; e < 8; e++) one(x[e], y[e], z[e], p[e], q[e]);
            if constexpr (!MAX) {
                *reinterpret_cast<uint4*>(dg + o + j * 8) = *reinterpret_cast<const uint4*>(p);
                *reinterpret_cast<uint4*>(du + o + j * 8) = *reinterpret_cast<const uint4*>(q);
            }
        } else {
            const uint32_t c0 = VEC ? j * 8 : j / 32 * 256 + j % 32;
            constexpr uint32_t step = VEC ? 1 : 32;
            T x[8], y[8], z[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; e++)
                if (c0 + e * step < a.F) {
                    x[e] = dhr[c0 + e * step];
                    y[e] = gr[c0 + e * step];
                    z[e] = ur[c0 + e * step];
                }
#pragma unroll
            for (uint32_t e = 0; e < 8; e++)
                if (c0 + e * step < a.F) one(x[e], y[e], z[e], dg[o + c0 + e * step], du[o + c0 + e * step]);
        }
    }
    if constexpr (MAX) {
        most = block_max(most);
        if (threadIdx.x == 0) a.part[blockIdx.x] = most;
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

// Where the operands of the tcgen05 product lie.
struct ForwardPlan {
    Operand2 x, wg, wu;
    size_t bytes;
};
ForwardPlan forward_plan(const vkblas_b200_gated_t& a, void* ws) {
    Carver c(ws);
    ForwardPlan p{};
    if (a.M > TOKENS_MAX) {
        p.x = operand(c, a.x, a.ldx, a.M, a.H);
        p.wg = operand(c, a.w_gate, a.ldwg, a.F, a.H);
        p.wu = operand(c, a.w_up, a.ldwu, a.F, a.H);
    }
    p.bytes = c.used;
    return p;
}

template <typename T> struct Forward {
    const vkblas_b200_gated_t& a;
    const ForwardPlan& f;
    const OpDevice& d;
    cudaStream_t s;
    template <int ACT, bool SAVE> cudaError_t go() const {
        return fused::launch_any<std::is_same<T, __nv_bfloat16>::value, GatedEpi<T, ACT, SAVE>>(
            a.M, a.F, a.H, fused::pick_half(a.M, a.F, true, d.num_sms), {f.x.p, f.x.ld}, {{f.wg.p, f.wg.ld}, {f.wu.p, f.wu.ld}},
            {fused::output(a.h, a.ldh, a.M, a.F), fused::output(a.g, a.ldg, a.M, a.F),
             fused::output(a.u, a.ldu, a.M, a.F)},
            d, s);
    }
    template <int ACT> cudaError_t operator()() const {
        cudaError_t e = fill(f.x, a.x, a.ldx, a.M, a.H, d.num_sms, s);
        if (e == cudaSuccess) e = fill(f.wg, a.w_gate, a.ldwg, a.F, a.H, d.num_sms, s);
        if (e == cudaSuccess) e = fill(f.wu, a.w_up, a.ldwu, a.F, a.H, d.num_sms, s);
        if (e != cudaSuccess) return e;
        return a.g ? go<ACT, true>() : go<ACT, false>();
    }
};

template <typename T>
cudaError_t forward(const vkblas_b200_gated_t& a, const ForwardPlan& f, const OpDevice& d, cudaStream_t s) {
    if (a.M > TOKENS_MAX) return by_act(a.act, Forward<T>{a, f, d, s});
    const TokenArgs t{a.x, a.w_gate, a.w_up, a.ldx, a.ldwg, a.ldwu, a.h, a.g, a.u, a.ldh, a.ldg, a.ldu, a.M, a.F, a.H};
    const bool vec = tma_readable(a.x, a.ldx) && tma_readable(a.w_gate, a.ldwg) && tma_readable(a.w_up, a.ldwu) &&
                     a.H % 8 == 0;
    return by_act(a.act, Token<T>{t, vec, d.num_sms, s});
}

// ------------------------------------------------------------- backward
// dG and dU go to the workspace; dx is one GEMM whose sum runs over both
// products, the weights' gradients are one GEMM each (umma_gemm.cu).
struct BackPlan {
    void *dg, *du;
    uint32_t ldo;
    Operand2 x, wg, wu;
    bool turn;                  // dU lies before dG
    float *part, *scale;        // GradArgs; null but for fp16
    uint32_t parts;             // room in part
    void* split;                // partial tiles of the GEMMs' last waves
    size_t bytes;
};
GemmProblem dx_problem(const vkblas_b200_gated_backward_t& a, const BackPlan& b) {
    GemmProblem p = product(a.dtype, 0, 0, a.M, a.H, 2 * ((a.F + 63) / 64 * 64), b.dg, b.ldo, b.wg.p, b.wg.ld, a.dx,
                            a.lddx);
    p.A2 = b.du, p.lda2 = b.ldo, p.B2 = b.wu.p, p.ldb2 = b.wu.ld, p.k1 = a.F;
    if (b.scale) p.d_alpha = b.scale, p.d_beta = b.scale + 1;
    return p;
}
// One weight's gradient, or (both) the two as a batch that shares X, where that takes
// fewer waves of tiles than one grid each.  The batch needs outputs of one leading
// dimension, a whole number of 16-byte units and at least a matrix apart.
bool dw_batched(const vkblas_b200_gated_backward_t& a) {
    const uint64_t tiles = (uint64_t)((a.F - 1) / 256 + 1) * ((a.H - 1) / 256 + 1), at_once = (uint64_t)op_num_sms() / 2;
    if ((2 * tiles - 1) / at_once + 1 >= 2 * ((tiles - 1) / at_once + 1)) return false;
    if (!a.dw_gate || !a.dw_up || a.lddwg != a.lddwu) return false;
    const uintptr_t g = reinterpret_cast<uintptr_t>(a.dw_gate), u = reinterpret_cast<uintptr_t>(a.dw_up);
    const uint64_t gap = g < u ? u - g : g - u;
    return gap % 16 == 0 && gap / 2 >= (uint64_t)a.F * a.lddwg && gap < (1ull << 40);
}
GemmProblem dw_problem(const vkblas_b200_gated_backward_t& a, const BackPlan& b, bool up, bool both) {
    if (both) up = b.turn;               // the first entry: the gradient at the lower address
    GemmProblem p = product(a.dtype, 1, 0, a.F, a.H, a.M, up ? b.du : b.dg, b.ldo, b.x.p, b.x.ld,
                            up ? a.dw_up : a.dw_gate, up ? a.lddwu : a.lddwg);
    if (b.scale) p.d_alpha = b.scale, p.d_beta = b.scale + 1;
    if (both) {
        p.batch = 2;
        p.sa = (int64_t)((size_t)a.M * b.ldo);
        p.sc = (static_cast<const char*>(up ? a.dw_gate : a.dw_up) - static_cast<const char*>(p.C)) / 2;
    }
    return p;
}
BackPlan back_plan(const vkblas_b200_gated_backward_t& a, void* ws) {
    Carver c(ws);
    BackPlan p{};
    p.ldo = up8(a.F);
    // dG and dU back to back (rows are whole 16-byte units), in the order in which their
    // weights' gradients lie, so that they are the two entries of a batch.
    const size_t one = (size_t)a.M * p.ldo;
    uint16_t* d = c.take<uint16_t>(2 * one);
    p.turn = reinterpret_cast<uintptr_t>(a.dw_up) < reinterpret_cast<uintptr_t>(a.dw_gate);
    p.dg = d ? d + (p.turn ? one : 0) : nullptr;
    p.du = d ? d + (p.turn ? 0 : one) : nullptr;
    if (a.dx) {
        p.wg = operand(c, a.w_gate, a.ldwg, a.F, a.H);
        p.wu = operand(c, a.w_up, a.ldwu, a.F, a.H);
    }
    if (a.dw_gate || a.dw_up) p.x = operand(c, a.x, a.ldx, a.M, a.H);
    const int sms = op_num_sms();
    if (a.dtype == VKBLAS_DT_F16) {
        p.parts = (uint32_t)sms * 8;
        p.part = c.take<float>(p.parts);
        p.scale = c.take<float>(2);
    }
    size_t split = a.dx ? umma_split_workspace_bytes(dx_problem(a, p), sms) : 0;
    if (a.dw_gate || a.dw_up)
        split = std::max(split, umma_split_workspace_bytes(dw_problem(a, p, false, dw_batched(a)), sms));
    p.split = c.take<char>(split);
    if (!split) p.split = nullptr;
    p.bytes = c.used;
    return p;
}

template <typename T> struct Grad {
    const GradArgs& g;
    bool vec;
    uint32_t blocks;
    cudaStream_t s;
    template <int ACT, bool VEC> cudaError_t go() const {
        if constexpr (std::is_same<T, __half>::value) {
            const cudaError_t e = launch_pdl(gated_grad_kernel<T, ACT, VEC, true>, g.parts, 256, s, g);
            if (e != cudaSuccess) return e;
        }
        return launch_pdl(gated_grad_kernel<T, ACT, VEC, false>, blocks, 256, s, g);
    }
    template <int ACT> cudaError_t operator()() const { return vec ? go<ACT, true>() : go<ACT, false>(); }
};

template <typename T>
cudaError_t backward(const vkblas_b200_gated_backward_t& a, const BackPlan& p, const OpDevice& d, cudaStream_t s) {
    cudaError_t e = cudaSuccess;
    if (a.dx) {
        e = fill(p.wg, a.w_gate, a.ldwg, a.F, a.H, d.num_sms, s);
        if (e == cudaSuccess) e = fill(p.wu, a.w_up, a.ldwu, a.F, a.H, d.num_sms, s);
    }
    if (e == cudaSuccess && (a.dw_gate || a.dw_up)) e = fill(p.x, a.x, a.ldx, a.M, a.H, d.num_sms, s);
    if (e != cudaSuccess) return e;
    const bool vec = tma_readable(a.dh, a.lddh) && tma_readable(a.g, a.ldg) && tma_readable(a.u, a.ldu);
    const uint64_t work = ((uint64_t)a.M * (vec ? (a.F + 7) / 8 : (a.F + 255) / 256 * 32) + 255) / 256, cap = (uint64_t)d.num_sms * 16;
    const GradArgs ga{a.dh, a.g, a.u, a.lddh, a.ldg, a.ldu, p.dg, p.du, p.ldo, a.M, a.F, p.part,
                      (uint32_t)std::min<uint64_t>(work, p.parts), p.scale};
    e = by_act(a.act, Grad<T>{ga, vec, (uint32_t)(work < cap ? work : cap), s});
    if (e == cudaSuccess && a.dx) e = launch_product(dx_problem(a, p), p.split, d, s);
    if (e == cudaSuccess && dw_batched(a)) return launch_product(dw_problem(a, p, false, true), p.split, d, s);
    if (e == cudaSuccess && a.dw_gate) e = launch_product(dw_problem(a, p, false, false), p.split, d, s);
    if (e == cudaSuccess && a.dw_up) e = launch_product(dw_problem(a, p, true, false), p.split, d, s);
    return e;
}

bool gated_ok(const vkblas_b200_gated_t* a) {
    return a && two_byte(a->dtype) && act_ok(a->act) && size_ok(a->M) && size_ok(a->F) && size_ok(a->H) &&
           mat_ok(a->x, a->ldx, a->H) && mat_ok(a->w_gate, a->ldwg, a->H) &&
           mat_ok(a->w_up, a->ldwu, a->H) && mat_ok(a->h, a->ldh, a->F) && !a->g == !a->u &&
           (!a->g || (mat_ok(a->g, a->ldg, a->F) && mat_ok(a->u, a->ldu, a->F)));
}

bool backward_ok(const vkblas_b200_gated_backward_t* a) {
    if (!a || !two_byte(a->dtype) || !act_ok(a->act) || !size_ok(a->M) || !size_ok(a->F) || !size_ok(a->H)) return false;
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

VKB_EXPORT size_t vkblas_b200_gated_workspace(const vkblas_b200_gated_t* a) {
    return gated_ok(a) ? forward_plan(*a, nullptr).bytes : 0;
}

VKB_EXPORT vkblas_status_t vkblas_b200_gated(const vkblas_b200_gated_t* a, void* workspace,
                                             size_t workspace_bytes, void* stream) {
    if (!gated_ok(a)) return VKBLAS_ERR_PARAM;
    const ForwardPlan f = forward_plan(*a, workspace);
    if (!ws_ok(workspace, workspace_bytes, f.bytes)) return VKBLAS_ERR_PARAM;
    OpDevice d;
    if (!op_device(&d)) return VKBLAS_ERR_INIT;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return op_status(a->dtype == VKBLAS_DT_F16 ? forward<__half>(*a, f, d, s) : forward<__nv_bfloat16>(*a, f, d, s));
}

VKB_EXPORT size_t vkblas_b200_gated_backward_workspace(const vkblas_b200_gated_backward_t* a) {
    return backward_ok(a) ? back_plan(*a, nullptr).bytes : 0;
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
    return op_status(a->dtype == VKBLAS_DT_F16 ? backward<__half>(*a, p, d, s)
                                               : backward<__nv_bfloat16>(*a, p, d, s));
}
