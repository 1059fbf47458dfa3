// xent.cu -- softmax cross entropy of a linear head, forward and backward,
// without keeping the logits.
//
//   z = X W^T (X T x H, W V x H), lse_i = log sum_j exp z_ij, loss_i = lse_i - z_i,t
//   D = diag(dloss) (exp(z - lse) - onehot(t)), dx = D W, dW = D^T X
#include <algorithm>
#include <type_traits>

#include "act.cuh"
#include "umma_fused.cuh"

namespace vkb {
namespace {

// e^(v - m) for v <= m, m finite; 0 for v = -inf.
__device__ __forceinline__ float exp_below(float v, float m) { return __expf(v - m); }
// The maximum a sum is taken relative to: 0 where the maximum is infinite, so
// that -inf - -inf never appears.
__device__ __forceinline__ float base_of(float m) { return isinf(m) ? 0.f : m; }

// Logits are summed in segments of SEG_KB k-blocks (512 products): the tensor core's own sum over
// all of K truncates (4.2e-6 of the logits at K = 4096), and losses and the gradients of well
// predicted tokens are small differences of what comes out.  Both passes take the same
// segments, so that exp(z - lse) sees the z that lse was made of.  Measured (1023 x 32000, K =
// 4096; error of the losses against 64 bits; step 4096 x 128000): segments of 256 220 us, 1.8e-7,
// 13.9 ms; 512 194 us, 3.6e-7, 13.1 ms; 1024 189 us, 7.6e-7, 13.1 ms; one of 4096 188 us, 3.2e-6,
// 13.0 ms; fp32 products of the library are 6.1e-7 off.
constexpr uint32_t SEG_KB = 8;

// This thread's half row (128 columns) of logits.  False when the CTA aborts.
template <typename A, typename R>
__device__ __forceinline__ bool half_row(const fused::Params& p, const fused::Tile& t, A&& acquire, R&& release,
                                         float (&z)[4][32]) {
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
        for (int i = 0; i < 32; i++) z[c][i] = -0.f;           // the identity of fp32 addition
    for (uint32_t kb = 0; kb < p.num_kb; kb += SEG_KB) {
        if (!acquire()) return false;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            uint32_t r[32];
            umma::tmem_ld_32x32b_x32(t.tmem + t.half * p.half + c * 32, r);
            umma::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i++) z[c][i] = __fadd_rn(z[c][i], __uint_as_float(r[i]));
        }
        release();
    }
    return true;
}

// Forward epilogue: each thread reduces its row's logits of half a tile (128) to their
// maximum and sum of exponentials, (m, s) with sum_j e^z_j = s e^base(m), and the
// thread whose columns hold the row's target stores that logit.  Nothing else of
// the T x V logits leaves the SM: 8 bytes a row and 128 columns do.
template <typename T>
struct StatsEpi {
    static constexpr uint32_t SEG_KB = vkb::SEG_KB;
    static constexpr bool TWO_B = false;
    struct Args {
        const int64_t* targets;
        float2* part;               // [2 tiles_n][T]
        float* zt;                  // [T]
    };
    template <typename A, typename R>
    static __device__ __forceinline__ void run(const fused::Params& p, const Args& a, const fused::Tile& t,
                                               A&& acquire, R&& release) {
        float z[4][32];
        if (!half_row(p, t, acquire, release, z)) return;
        const uint32_t n0 = (2 * t.nb + t.half) * p.half;
        const uint32_t cols = n0 < p.N ? min(p.half, p.N - n0) : 0;
        const bool row = t.m < p.M;
        if (cols < 128) {                                       // past the half or the vocabulary: no term
#pragma unroll
            for (int c = 0; c < 4; c++)
#pragma unroll
                for (int i = 0; i < 32; i++)
                    if (c * 32 + i >= cols) z[c][i] = -INFINITY;
        }
        const int64_t tg = row ? a.targets[t.m] - (int64_t)n0 : -1;
        if (__any_sync(~0u, tg >= 0 && tg < cols)) {
            float v = 0.f;
#pragma unroll
            for (int c = 0; c < 4; c++)
#pragma unroll
                for (int i = 0; i < 32; i++)
                    if (tg == c * 32 + i) v = z[c][i];
            if (tg >= 0 && tg < cols) a.zt[t.m] = v;
        }
        float m = z[0][0];
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int i = 0; i < 32; i++) m = fmaxf(m, z[c][i]);
        const float base = base_of(m);
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int i = 0; i < 32; i++) s[i & 3] += exp_below(z[c][i], base);
        if (row) a.part[(size_t)(2 * t.nb + t.half) * p.M + t.m] = make_float2(m, (s[0] + s[1]) + (s[2] + s[3]));
    }
};

// (m, s) of two sets of logits together.  An empty set is (-inf, 0).
__device__ __forceinline__ float2 join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x), base = base_of(m);
    const float sa = a.y == 0.f ? 0.f : a.y * __expf(base_of(a.x) - base);
    const float sb = b.y == 0.f ? 0.f : b.y * __expf(base_of(b.x) - base);
    return make_float2(m, sa + sb);
}

// Joins the partial sums of 32 rows: warp w of 32 takes every 32nd partial (lanes are
// rows, so loads are coalesced), then warp 0 joins the 32 results in order.
__global__ void __launch_bounds__(1024) xent_finish_kernel(const float2* part, const float* zt, uint32_t parts, uint32_t T,
                                                           const int64_t* targets, int64_t ignore, int64_t V, float* loss,
                                                           float* lse) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ float2 sh[32][33];
    const uint32_t lane = threadIdx.x & 31, w = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
    float2 acc = make_float2(-INFINITY, 0.f);
    if (i < T) {
        uint32_t j = w;
        for (; j + 96 < parts; j += 128) {
            float2 v[4];
#pragma unroll
            for (int q = 0; q < 4; q++) v[q] = part[(size_t)(j + 32 * q) * T + i];
#pragma unroll
            for (int q = 0; q < 4; q++) acc = join(acc, v[q]);
        }
        for (; j < parts; j += 32) acc = join(acc, part[(size_t)j * T + i]);
    }
    sh[w][lane] = acc;
    __syncthreads();
    if (w != 0 || i >= T) return;
    for (uint32_t j = 1; j < 32; j++) acc = join(acc, sh[j][lane]);
    const float l = base_of(acc.x) + logf(acc.y);
    if (lse) lse[i] = l;
    const int64_t t = targets[i];
    loss[i] = t == ignore ? 0.f : t < 0 || t >= V ? NAN : l - zt[i];
}

// Backward epilogue: D = coef (exp(z - lse) - onehot) of a piece of the vocabulary,
// rounded to the operand type and stored for the two products that read it.  coef is
// S dloss: S brings the largest |dloss| to [2^14, 2^15), so that in fp16, too, a
// probability of 1e-8 is a normal number; the products divide by S in fp32.  The target's
// entry is expm1(z - lse), and z - lse is one subtraction: where the target has most of the
// probability, what is left of it is as good as lse (2^-24 of its size).
template <typename T>
struct GradEpi {
    static constexpr uint32_t SEG_KB = vkb::SEG_KB;
    static constexpr bool TWO_B = false;
    struct Args {
        const int64_t* targets;
        int64_t ignore, V, first;   // first: the piece's first column
        const float *dloss, *lse, *scale;
        fused::Out d;
    };
    template <typename A, typename R>
    static __device__ __forceinline__ void run(const fused::Params& p, const Args& a, const fused::Tile& t,
                                               A&& acquire, R&& release) {
        const uint32_t n0 = (2 * t.nb + t.half) * p.half;
        float coef = 0.f, lse = 0.f;
        int tg = -1;                             // the target's column among this warp's
        bool kept = false;
        if (t.m < p.M) {
            const int64_t y = a.targets[t.m], at = y - a.first - (int64_t)n0;
            kept = y != a.ignore;
            coef = y < 0 || y >= a.V ? NAN : a.dloss[t.m] * a.scale[0];
            lse = a.lse[t.m];
            if (at >= 0 && at < p.half) tg = (int)at;
        }
        float z[4][32];
        if (!half_row(p, t, acquire, release, z)) return;
        uint32_t d[2][32];
#pragma unroll
        for (int c = 0; c < 4; c++) {
            float zt = 0.f;
#pragma unroll
            for (int i = 0; i < 32; i++) {
                const float v = z[c][i] - lse;
                if (tg == c * 32 + i) zt = v;
                z[c][i] = fast_exp2(v * LOG2E);
            }
            if (__any_sync(~0u, tg >= 32 * c && tg < 32 * c + 32)) {       // seldom
                const float e = expm1f(zt);
#pragma unroll
                for (int i = 0; i < 32; i++)
                    if (tg == c * 32 + i) z[c][i] = e;
            }
#pragma unroll
            for (int i = 0; i < 16; i++)
                d[c >> 1][(c & 1) * 16 + i] = fused::pack2<T>(coef * z[c][2 * i], coef * z[c][2 * i + 1]);
        }
        // An ignored row's x may hold anything: its D is 0, not coef * p.
#pragma unroll
        for (int i = 0; i < 32; i++) d[0][i] = kept ? d[0][i] : 0u, d[1][i] = kept ? d[1][i] : 0u;
#pragma unroll
        for (uint32_t h = 0; h < 2; h++)
            if (h * 64 < p.half) fused::store_rows(a.d, t, n0 + h * 64, min(64u, p.half - h * 64), d[h]);
    }
};

// Before the pieces, in one launch.  Block 0: out[0] = S, out[1] = 1 / S, out[2] = 0 (beta
// of the products), S the power of two that brings the largest |dloss| of a kept row
// into [2^14, 2^15).  The others (where xk): X with the ignored rows cleared, in rows of
// ld (a multiple of 8), so that D^T X does not see whatever a padding token's row holds.
template <typename T>
__global__ void __launch_bounds__(256) xent_prepare_kernel(const float* dloss, const int64_t* t, int64_t ignore, uint32_t rows,
                                                           float* out, const uint16_t* x, uint32_t ldx, uint32_t H, bool vec,
                                                           uint16_t* xk, uint32_t ld) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (blockIdx.x == 0) {
        __shared__ float sm[8];
        float m = 0.f;
        for (uint32_t i = threadIdx.x; i < rows; i += 256) {
            const float v = dloss[i];
            if (t[i] != ignore && isfinite(v)) m = fmaxf(m, fabsf(v));
        }
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = m;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < 8; w++) m = fmaxf(m, sm[w]);
            const int e = m > 0.f ? max(ilogbf(m), -100) : 14;
            out[0] = scalbnf(1.f, 14 - e);
            out[1] = scalbnf(1.f, e - 14);
            out[2] = 0.f;
        }
        return;
    }
    const uint32_t per = ld / 8;
    const uint64_t total = (uint64_t)rows * per, stride = (uint64_t)(gridDim.x - 1) * 256;
    for (uint64_t i = (uint64_t)(blockIdx.x - 1) * 256 + threadIdx.x; i < total; i += stride) {
        const uint32_t r = (uint32_t)(i / per), c = (uint32_t)(i - (uint64_t)r * per) * 8;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (t[r] != ignore) {
            const uint16_t* p = x + (size_t)r * ldx + c;
            v = vec && c + 8 <= H ? ld16(p) : gather8(p, (int64_t)H - c);
        }
        *reinterpret_cast<uint4*>(xk + (size_t)r * ld + c) = v;
    }
}

// dx = acc / S, rounded to the operand type.
template <typename T>
__global__ void __launch_bounds__(256) store_dx_kernel(const float* acc, uint32_t rows, uint32_t H, uint32_t lda,
                                                       const float* scale, T* dx, uint32_t ld) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float inv = scale[1];
    const uint32_t per = (H + 3) / 4;                        // lda is a multiple of 4
    const uint64_t total = (uint64_t)rows * per;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
        const uint32_t r = (uint32_t)(i / per), c = (uint32_t)(i - (uint64_t)r * per) * 4;
        const float4 v = __ldcs(reinterpret_cast<const float4*>(acc + (size_t)r * lda + c));
        const T e[4] = {Elem<T>::from_f(v.x * inv), Elem<T>::from_f(v.y * inv), Elem<T>::from_f(v.z * inv),
                        Elem<T>::from_f(v.w * inv)};
        T* o = dx + (size_t)r * ld + c;
        if (c + 4 <= H && (reinterpret_cast<uintptr_t>(o) & 7u) == 0)
            *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(e);
        else
            for (uint32_t j = 0; j < 4 && c + j < H; j++) o[j] = e[j];
    }
}

bool xent_ok(const vkblas_b200_linear_xent_t* a) {
    return a && two_byte(a->dtype) && size_ok(a->T) && size_ok(a->V) && size_ok(a->H) && mat_ok(a->x, a->ldx, a->H) &&
           mat_ok(a->w, a->ldw, a->H) && a->targets && is_al(a->targets, 8) && a->loss &&
           is_al(a->loss, 4) && is_al(a->lse, 4);
}
bool backward_ok(const vkblas_b200_linear_xent_backward_t* a) {
    return a && two_byte(a->dtype) && size_ok(a->T) && size_ok(a->V) && size_ok(a->H) && mat_ok(a->x, a->ldx, a->H) &&
           mat_ok(a->w, a->ldw, a->H) && a->targets && is_al(a->targets, 8) && a->dloss &&
           is_al(a->dloss, 4) && a->lse && is_al(a->lse, 4) && (a->dx || a->dw) &&
           (!a->dx || mat_ok(a->dx, a->lddx, a->H)) && (!a->dw || mat_ok(a->dw, a->lddw, a->H));
}

struct FwdPlan {
    Operand2 x, w;
    float2* part;
    float* zt;
    uint32_t half, parts;
    size_t bytes;
};
FwdPlan fwd_plan(const vkblas_b200_linear_xent_t& a, void* ws) {
    Carver c(ws);
    FwdPlan p;
    p.x = operand(c, a.x, a.ldx, a.T, a.H);
    p.w = operand(c, a.w, a.ldw, a.V, a.H);
    p.half = fused::pick_half(a.T, a.V, false, op_num_sms());
    p.parts = 2 * ((a.V - 1) / (2 * p.half) + 1);
    p.part = c.take<float2>((size_t)p.parts * a.T);
    p.zt = c.take<float>(a.T);
    p.bytes = c.used;
    return p;
}

// The backward pass goes over the vocabulary in pieces of equal width, so that D takes
// at most about PIECE_BYTES, but no fewer than PIECE_TILES x 256 columns: each piece is
// three large products, and adds to dx in memory once.
constexpr size_t PIECE_BYTES = 256u << 20;
constexpr uint64_t PIECE_TILES = 32;
// Columns that dx = D W may sum in one accumulator.  The tensor core cuts what it adds at the
// accumulator's last place, so a sum of one sign comes out too small by about 1e-8 of it
// for each column (1023 x 131072, K = 4096, weights of one sign: 5.3e-4 in one sum, 2.6e-4 to
// 3.2e-4 in sums of 32768, 9e-5 in sums of 8192).  Half a rounding step is 4.9e-4 in fp16
// and 3.9e-3 in bf16; the sums stay below a quarter of that, and are added up in fp32.
inline uint32_t max_sum(int dtype) { return dtype == VKBLAS_DT_F16 ? 8192 : 65536; }

struct BwdPlan {
    Operand2 x, w;
    uint32_t pieces, width;      // columns a piece (a multiple of 256); D's row stride
    uint32_t part;               // columns of a piece that one product for dx takes (the same)
    void* d;
    void* xk;                    // X with the ignored rows cleared
    uint32_t ldk, lda;
    float *acc, *scale;
    void* split;
    size_t bytes;
};
inline bool dx_summed(const BwdPlan& b) { return b.pieces > 1 || b.part < b.width; }
// The products of the piece from column `first`: dx of its n columns from `at`, dW of n.
template <typename P>
GemmProblem dx_problem(const P& a, const BwdPlan& b, uint64_t first, uint32_t at, uint32_t n) {
    const uint16_t *w = static_cast<const uint16_t*>(b.w.p), *d = static_cast<const uint16_t*>(b.d);
    const bool sum = dx_summed(b);
    GemmProblem p = product(a.dtype, 0, 0, a.T, a.H, n, d ? d + at : d, b.width, w ? w + (first + at) * b.w.ld : w,
                            b.w.ld, sum ? static_cast<void*>(b.acc) : a.dx, sum ? b.lda : a.lddx);
    if (sum) {                   // fp32 sum over the products
        p.c_f32 = true;
        p.beta = first + at ? 1.f : 0.f;
    } else if (b.scale) {
        p.d_alpha = b.scale + 1;
        p.d_beta = b.scale + 2;
    }
    return p;
}
template <typename P>
GemmProblem dw_problem(const P& a, const BwdPlan& b, uint64_t first, uint32_t n) {
    GemmProblem p = product(a.dtype, 1, 0, n, a.H, a.T, b.d, b.width, b.xk, b.ldk,
                            a.dw ? static_cast<uint16_t*>(a.dw) + first * a.lddw : nullptr, a.lddw);
    if (b.scale) {
        p.d_alpha = b.scale + 1;
        p.d_beta = b.scale + 2;
    }
    return p;
}
BwdPlan bwd_plan(const vkblas_b200_linear_xent_backward_t& a, void* ws) {
    Carver c(ws);
    BwdPlan p{};
    const uint64_t tiles = (a.V - 1) / fused::BN + 1;
    const uint64_t fit = std::max(PIECE_TILES, PIECE_BYTES / 2 / a.T / fused::BN);
    p.pieces = (uint32_t)((tiles - 1) / fit + 1);
    p.width = (uint32_t)((tiles - 1) / p.pieces + 1) * fused::BN;
    p.pieces = (uint32_t)((a.V - 1) / p.width + 1);
    p.x = operand(c, a.x, a.ldx, a.T, a.H);
    p.w = operand(c, a.w, a.ldw, a.V, a.H);
    p.d = c.take<uint16_t>((size_t)a.T * p.width);
    p.ldk = up8(a.H);
    p.xk = c.take<uint16_t>(a.dw ? (size_t)a.T * p.ldk : 0);
    p.lda = up8(a.H);
    const int sms = op_num_sms();
    // As few products for dx as keep each accumulator's share of K within max_sum (a product of
    // few tiles is cut along K as it is).
    p.part = p.width;
    for (uint32_t parts = 1; a.dx; parts++) {
        p.part = ((p.width - 1) / parts / fused::BN + 1) * fused::BN;
        const UmmaPlan u = umma_plan(dx_problem(a, p, 0, 0, std::min(p.part, a.V)), sms, false);
        const uint64_t longest = 64ull * (u.splits > 1 && u.full_tiles == 0 ? u.kblocks_per_split : u.kblocks);
        if (longest <= max_sum(a.dtype)) break;
    }
    p.acc = c.take<float>(a.dx && dx_summed(p) ? (size_t)a.T * p.lda : 0);
    p.scale = c.take<float>(3);
    const uint32_t last = (uint32_t)(a.V - (uint64_t)(p.pieces - 1) * p.width);
    size_t split = 0;
    for (uint32_t n : {std::min(p.width, a.V), last}) {
        if (a.dx)
            for (uint32_t k : {std::min(p.part, n), (n - 1) % p.part + 1})
                split = std::max(split, umma_split_workspace_bytes(dx_problem(a, p, 0, 0, k), sms));
        if (a.dw) split = std::max(split, umma_split_workspace_bytes(dw_problem(a, p, 0, n), sms));
    }
    p.split = c.take<char>(split);
    if (!split) p.split = nullptr;
    p.bytes = c.used;
    return p;
}

template <typename T> constexpr bool is_bf16() { return std::is_same<T, __nv_bfloat16>::value; }

template <typename T>
cudaError_t forward(const vkblas_b200_linear_xent_t& a, const FwdPlan& f, const OpDevice& d, cudaStream_t s) {
    cudaError_t e = fill(f.x, a.x, a.ldx, a.T, a.H, d.num_sms, s);
    if (e == cudaSuccess) e = fill(f.w, a.w, a.ldw, a.V, a.H, d.num_sms, s);
    if (e == cudaSuccess)
        e = fused::launch_any<is_bf16<T>(), StatsEpi<T>>(a.T, a.V, a.H, f.half, {f.x.p, f.x.ld}, {{f.w.p, f.w.ld}, {}},
                                                         {a.targets, f.part, f.zt}, d, s);
    if (e != cudaSuccess) return e;
    return launch_pdl(xent_finish_kernel, (a.T - 1) / 32 + 1, 1024, s, static_cast<const float2*>(f.part),
                      static_cast<const float*>(f.zt), f.parts, a.T, a.targets, a.ignore_index, (int64_t)a.V, a.loss, a.lse);
}

template <typename T>
cudaError_t backward(const vkblas_b200_linear_xent_backward_t& a, const BwdPlan& b, const OpDevice& d, cudaStream_t s) {
    cudaError_t e = fill(b.x, a.x, a.ldx, a.T, a.H, d.num_sms, s);
    if (e == cudaSuccess) e = fill(b.w, a.w, a.ldw, a.V, a.H, d.num_sms, s);
    if (e != cudaSuccess) return e;
    const uint64_t groups = a.dw ? ((uint64_t)a.T * (b.ldk / 8) + 255) / 256 : 0;
    e = launch_pdl(xent_prepare_kernel<T>, 1 + (uint32_t)std::min<uint64_t>(groups, d.num_sms * 16), 256, s, a.dloss, a.targets,
                   a.ignore_index, a.T, b.scale, static_cast<const uint16_t*>(a.x), a.ldx, a.H, tma_readable(a.x, a.ldx),
                   static_cast<uint16_t*>(b.xk), b.ldk);
    if (e != cudaSuccess) return e;
    for (uint64_t f = 0; f < a.V; f += b.width) {
        const uint32_t n = (uint32_t)std::min<uint64_t>(b.width, a.V - f);
        const fused::Matrix w{static_cast<const T*>(b.w.p) + f * b.w.ld, b.w.ld};
        e = fused::launch_any<is_bf16<T>(), GradEpi<T>>(
            a.T, n, a.H, fused::pick_half(a.T, n, false, d.num_sms), {b.x.p, b.x.ld}, {w, {}},
            {a.targets, a.ignore_index, a.V, (int64_t)f, a.dloss, a.lse, b.scale, fused::output(b.d, b.width, a.T, n)}, d, s);
        for (uint32_t k = 0; e == cudaSuccess && a.dx && k < n; k += b.part)
            e = launch_product(dx_problem(a, b, f, k, std::min(b.part, n - k)), b.split, d, s);
        if (e == cudaSuccess && a.dw) e = launch_product(dw_problem(a, b, f, n), b.split, d, s);
        if (e != cudaSuccess) return e;
    }
    if (a.dx && dx_summed(b))
        e = launch_pdl(store_dx_kernel<T>, d.num_sms * 8, 256, s, static_cast<const float*>(b.acc), a.T, a.H, b.lda,
                       static_cast<const float*>(b.scale), static_cast<T*>(a.dx), a.lddx);
    return e;
}

}  // namespace
}  // namespace vkb

using namespace vkb;
#define VKB_EXPORT extern "C" __attribute__((visibility("default")))

VKB_EXPORT size_t vkblas_b200_linear_xent_workspace(const vkblas_b200_linear_xent_t* a) {
    return xent_ok(a) ? fwd_plan(*a, nullptr).bytes : 0;
}

VKB_EXPORT vkblas_status_t vkblas_b200_linear_xent(const vkblas_b200_linear_xent_t* a, void* workspace,
                                                   size_t workspace_bytes, void* stream) {
    if (!xent_ok(a)) return VKBLAS_ERR_PARAM;
    const FwdPlan p = fwd_plan(*a, workspace);
    if (!ws_ok(workspace, workspace_bytes, p.bytes)) return VKBLAS_ERR_PARAM;
    OpDevice d;
    if (!op_device(&d)) return VKBLAS_ERR_INIT;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return op_status(a->dtype == VKBLAS_DT_F16 ? forward<__half>(*a, p, d, s) : forward<__nv_bfloat16>(*a, p, d, s));
}

VKB_EXPORT size_t vkblas_b200_linear_xent_backward_workspace(const vkblas_b200_linear_xent_backward_t* a) {
    return backward_ok(a) ? bwd_plan(*a, nullptr).bytes : 0;
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
    return op_status(a->dtype == VKBLAS_DT_F16 ? backward<__half>(*a, p, d, s) : backward<__nv_bfloat16>(*a, p, d, s));
}
