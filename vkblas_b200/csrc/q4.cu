// q4.cu -- decode products with 4-bit weights and group scales.
//
//   y[m, n] = alpha * sum_k x[m, k] * s[n, k/G] * (q[n, k] - z[n, k/G]) + beta * y[m, n]
//
// One pass over N K / 2 bytes of weights, bound by memory for one token; for more
// the conversion of the weights shares the time.  Per group G the products of the
// integers q - z (exact in both 2-byte types) are summed on the tensor cores, and
// that sum times the scale is added to an fp32 sum, so neither the scale nor a
// product is rounded to 2 bytes.
//
// Packed form, written once by vkblas_b200_q4_pack: blocks of 16 weight rows, and in
// a block steps of 128 k.  A step is 1024 bytes: lane l = 4 g + t of a warp reads 16
// bytes of row g and 16 of row g + 8 (two fully coalesced 512-byte loads).  Word w of
// the 16 bytes holds k = 32 w + 8 t + 0..7, so that a word's MMAs lie in one run of 32
// k, whatever multiple of 32 the group is; its nibble i < 4 is k = 2 i and nibble 4 + i
// is k = 2 i + 1, so that one mask yields a pair of neighbours for the MMA.  Scales
// (and zero points, a byte each) follow as [block][group][16 rows].
#include "ops.cuh"

namespace vkb {
namespace {

constexpr uint32_t ROWS = 16, STEP = 128, STEP_BYTES = 1024;

struct Layout {
    uint32_t blocks, steps, ng;
    size_t scales, zeros, bytes;
};
Layout layout(const vkblas_b200_q4_t& w) {
    Layout l;
    l.blocks = (w.N - 1) / ROWS + 1;
    l.steps = (w.K - 1) / STEP + 1;
    l.ng = (w.K - 1) / w.group + 1;
    l.scales = (size_t)l.blocks * l.steps * STEP_BYTES;
    l.zeros = l.scales + up256((size_t)l.blocks * l.ng * ROWS * 2);
    l.bytes = l.zeros + (w.has_zeros ? up256((size_t)l.blocks * l.ng * ROWS) : 0);
    return l;
}

// One thread per packed word, then per scale.  Rows past N and k past K are zeros
// (with scale 0).
__global__ void __launch_bounds__(256) q4_pack_kernel(uint32_t N, uint32_t K, Layout l, const uint8_t* q, uint32_t ldq,
                                                      const uint16_t* s, uint32_t lds, const uint8_t* z, uint32_t ldz,
                                                      uint8_t* out) {
    const uint64_t first = (uint64_t)blockIdx.x * 256 + threadIdx.x, stride = (uint64_t)gridDim.x * 256;
    const uint64_t words = (uint64_t)l.blocks * l.steps * (STEP_BYTES / 4);
    for (uint64_t i = first; i < words; i += stride) {
        const uint32_t in = (uint32_t)(i % 256);                 // word of the step: [half][lane][w]
        const uint64_t bs = i / 256;
        const uint32_t w = in & 3, lane = (in >> 2) & 31, half = in >> 7;
        const uint64_t n = bs / l.steps * ROWS + (lane >> 2) + 8 * half;
        const uint64_t k = bs % l.steps * STEP + 32 * w + 8 * (lane & 3);
        uint32_t v = 0;
        if (n < N) {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++)
                if (k + j < K) {
                    const uint32_t nib = (q[n * ldq + (k + j) / 2] >> (4 * (j & 1))) & 15u;
                    v |= nib << (4 * ((j & 1) * 4 + (j >> 1)));
                }
        }
        reinterpret_cast<uint32_t*>(out)[i] = v;
    }
    const uint64_t cells = (uint64_t)l.blocks * l.ng * ROWS;
    for (uint64_t i = first; i < cells; i += stride) {
        const uint64_t bg = i / ROWS, n = bg / l.ng * ROWS + i % ROWS, g = bg % l.ng;
        reinterpret_cast<uint16_t*>(out + l.scales)[i] = n < N ? s[n * lds + g] : (uint16_t)0;
        if (z) out[l.zeros + i] = n < N ? z[n * ldz + g] & 15 : 0;
    }
}

// The type's half of the conversion.  A nibble OR-ed into the mantissa of MAGIC (1024
// in fp16, 128 in bf16) is MAGIC + q exactly, and subtracting MAGIC + z leaves q - z
// exactly.  fp16 has room for the nibble four bits higher, too: 1024 + 16 q, which one
// FMA turns into q - z, and saves two of the three shifts a word.
template <typename T> struct Dec;
template <> struct Dec<__half> {
    using Pair = __half2;
    Pair lo, hi;                       // 1024 + z and -(64 + z), twice
    __device__ __forceinline__ void set(uint32_t z) {
        lo = __half2half2(__ushort_as_half((unsigned short)(0x6400u + z)));
        hi = __half2half2(__ushort_as_half((unsigned short)(0xD400u + (z << 4))));
    }
    static __device__ __forceinline__ Pair mask(uint32_t v, uint32_t m) {
        const uint32_t r = (v & m) | 0x64006400u;
        return *reinterpret_cast<const Pair*>(&r);
    }
    __device__ __forceinline__ void run(uint32_t v, uint32_t (&p)[4]) const {
        const Pair sixteenth = __half2half2(__ushort_as_half((unsigned short)0x2C00u));
        Pair d[4];
        d[0] = __hsub2(mask(v, 0x000F000Fu), lo);
        d[1] = __hfma2(mask(v, 0x00F000F0u), sixteenth, hi);
        v >>= 8;
        d[2] = __hsub2(mask(v, 0x000F000Fu), lo);
        d[3] = __hfma2(mask(v, 0x00F000F0u), sixteenth, hi);
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = *reinterpret_cast<const uint32_t*>(&d[i]);
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Dec<__nv_bfloat16> {
    using Pair = __nv_bfloat162;
    Pair lo;                           // 128 + z, twice
    __device__ __forceinline__ void set(uint32_t z) {
        lo = __bfloat162bfloat162(__ushort_as_bfloat16((unsigned short)(0x4300u + z)));
    }
    __device__ __forceinline__ void run(uint32_t v, uint32_t (&p)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t r = ((v >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
            const Pair d = __hsub2(*reinterpret_cast<const Pair*>(&r), lo);
            p[i] = *reinterpret_cast<const uint32_t*>(&d);
        }
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

struct Args {
    const uint8_t* w;
    Layout l;
    uint32_t M, N, K, group;
    const uint16_t* x;
    uint32_t ldx;
    void* y;
    uint32_t ldy;
    float alpha, beta;
};

__device__ __forceinline__ uint4 ldg_weights(const uint8_t* p) {
    uint4 v;
    asm("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
        : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Eight activations from element offset k of a row, zeros past K.  AL: elements that a
// row's start and k are aligned to (8, 4, 2 or 1).
template <int AL>
__device__ __forceinline__ uint4 load_x(const uint16_t* p, uint32_t k, uint32_t K, bool ok) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (!ok || k >= K) return v;
    if (AL > 1 && k + 8 <= K) {
        if constexpr (AL == 8) {
            v = __ldg(reinterpret_cast<const uint4*>(p + k));
        } else if constexpr (AL == 4) {
            const uint2 a = __ldg(reinterpret_cast<const uint2*>(p + k)), b = __ldg(reinterpret_cast<const uint2*>(p + k) + 1);
            v = make_uint4(a.x, a.y, b.x, b.y);
        } else {
            const uint32_t* q = reinterpret_cast<const uint32_t*>(p + k);
            v = make_uint4(__ldg(q), __ldg(q + 1), __ldg(q + 2), __ldg(q + 3));
        }
    } else {
        uint32_t e[8];
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = k + i < K ? (uint32_t)__ldg(p + k + i) : 0u;
        v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
    }
    return v;
}

// A CTA owns 16 weight rows; its KW warps take contiguous runs of 128-k steps and add
// their sums through shared memory in warp order.  UN steps' weights are loaded
// together, so that a lane has 2 UN 128-bit loads in flight.
template <typename T, bool TWO, bool ZEROS, int AL, int KW>
__global__ void __launch_bounds__(KW * 32) q4_gemv_kernel(const Args a) {
    constexpr uint32_t UN = TWO ? 2 : 4;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t b = blockIdx.x, per = (a.l.steps + KW - 1) / KW;
    const uint32_t s0 = min(a.l.steps, warp * per), s1 = min(a.l.steps, s0 + per);
    const uint8_t* wp = a.w + (size_t)b * a.l.steps * STEP_BYTES + lane * 16;
    const T* sp = reinterpret_cast<const T*>(a.w + a.l.scales) + (size_t)b * a.l.ng * ROWS + g;
    const uint8_t* zp = a.w + a.l.zeros + (size_t)b * a.l.ng * ROWS + g;
    const bool x0ok = g < a.M, x1ok = TWO && g + 8 < a.M;
    const uint16_t* x0 = a.x + (size_t)(x0ok ? g : 0) * a.ldx;
    const uint16_t* x1 = a.x + (size_t)(x1ok ? g + 8 : 0) * a.ldx;

    constexpr int NT = TWO ? 2 : 1;
    float sum[NT][4], d[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) sum[n][i] = d[n][i] = 0.f;
    // The group in progress and its scales; every 32 k may start the next one.
    uint32_t grp = s0 * STEP / a.group, gend = (grp + 1) * a.group;
    float sc0 = 0.f, sc1 = 0.f;
    Dec<T> z0, z1;
    z0.set(8);
    z1.set(8);
    auto open = [&]() {
        sc0 = Elem<T>::to_f(sp[(size_t)grp * ROWS]);
        sc1 = Elem<T>::to_f(sp[(size_t)grp * ROWS + 8]);
        if constexpr (ZEROS) {
            z0.set(zp[(size_t)grp * ROWS]);
            z1.set(zp[(size_t)grp * ROWS + 8]);
        }
    };
    auto close = [&]() {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                sum[n][i] = fmaf(i < 2 ? sc0 : sc1, d[n][i], sum[n][i]);
                d[n][i] = 0.f;
            }
    };
    if (s0 < s1) open();
    for (uint32_t s = s0; s < s1; s += UN) {
        uint4 w[UN][2];
#pragma unroll
        for (uint32_t j = 0; j < UN; j++) {
            const uint8_t* p = wp + (size_t)min(s + j, s1 - 1) * STEP_BYTES;
            w[j][0] = ldg_weights(p);
            w[j][1] = ldg_weights(p + 512);
        }
#pragma unroll
        for (uint32_t j = 0; j < UN; j++) {
            if (s + j >= s1) break;
            const uint32_t* lo = reinterpret_cast<const uint32_t*>(&w[j][0]);
            const uint32_t* hi = reinterpret_cast<const uint32_t*>(&w[j][1]);
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const uint32_t kb = (s + j) * STEP + 32 * i;
                if (kb >= gend && kb < a.K) {
                    close();
                    grp++;
                    gend += a.group;
                    open();
                }
                uint32_t p0[4], p1[4];
                z0.run(lo[i], p0);
                z1.run(hi[i], p1);
                const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]}, a1[4] = {p0[2], p1[2], p0[3], p1[3]};
                const uint4 xa = load_x<AL>(x0, kb + 8 * t, a.K, x0ok);
                Dec<T>::mma(d[0], a0, xa.x, xa.y);
                Dec<T>::mma(d[0], a1, xa.z, xa.w);
                if constexpr (TWO) {
                    const uint4 xb = load_x<AL>(x1, kb + 8 * t, a.K, x1ok);
                    Dec<T>::mma(d[1], a0, xb.x, xb.y);
                    Dec<T>::mma(d[1], a1, xb.z, xb.w);
                }
            }
        }
    }
    close();

    __shared__ float red[KW][NT * 4][32];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) red[warp][4 * n + i][lane] = sum[n][i];
    __syncthreads();
    // Warp n adds tokens 8 n .. 8 n + 7.  Fragment: (row g, tokens 2t, 2t + 1), (row g + 8, the same).
    if (warp >= NT) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float v = red[0][4 * warp + i][lane];
#pragma unroll
        for (int w = 1; w < KW; w++) v = __fadd_rn(v, red[w][4 * warp + i][lane]);
        const uint32_t n = b * ROWS + g + (i < 2 ? 0 : 8), m = 8 * warp + 2 * t + (i & 1);
        if (n < a.N && m < a.M) {
            T* y = static_cast<T*>(a.y) + (size_t)m * a.ldy + n;
            *y = Elem<T>::from_f(epilogue(a.alpha, v, a.beta, a.beta != 0.f ? Elem<T>::to_f(*y) : 0.f));
        }
    }
}

template <typename T, bool TWO, bool ZEROS, int AL>
void launch_kw(const Args& a, int kw, cudaStream_t s) {
    if (kw == 4) q4_gemv_kernel<T, TWO, ZEROS, AL, 4><<<a.l.blocks, 128, 0, s>>>(a);
    else if (kw == 8) q4_gemv_kernel<T, TWO, ZEROS, AL, 8><<<a.l.blocks, 256, 0, s>>>(a);
    else q4_gemv_kernel<T, TWO, ZEROS, AL, 16><<<a.l.blocks, 512, 0, s>>>(a);
}
template <typename T, bool TWO, bool ZEROS>
void launch_al(const Args& a, int kw, cudaStream_t s) {
    const size_t bits = reinterpret_cast<uintptr_t>(a.x) / 2 | (a.M > 1 ? a.ldx : 0);   // in elements
    if (bits % 8 == 0) launch_kw<T, TWO, ZEROS, 8>(a, kw, s);
    else if (bits % 4 == 0) launch_kw<T, TWO, ZEROS, 4>(a, kw, s);
    else if (bits % 2 == 0) launch_kw<T, TWO, ZEROS, 2>(a, kw, s);
    else launch_kw<T, TWO, ZEROS, 1>(a, kw, s);
}
template <typename T>
cudaError_t launch_q4(const Args& a, bool zeros, int num_sms, cudaStream_t s) {
    // Warps a CTA: enough that all SMs together hold about 24 warps each, but not more
    // than one a step of 128 k.
    int kw = 4;
    while (kw < 16 && (uint64_t)a.l.blocks * kw < 24ull * num_sms && a.l.steps >= 2u * kw) kw *= 2;
    const bool two = a.M > 8;
    if (two) zeros ? launch_al<T, true, true>(a, kw, s) : launch_al<T, true, false>(a, kw, s);
    else zeros ? launch_al<T, false, true>(a, kw, s) : launch_al<T, false, false>(a, kw, s);
    count_launch();
    return cudaGetLastError();
}

bool q4_ok(const vkblas_b200_q4_t* w) {
    return w && two_byte(w->dtype) && size_ok(w->N) && size_ok(w->K) && w->group % 32 == 0 && size_ok(w->group);
}

}  // namespace
}  // namespace vkb

using namespace vkb;
#define VKB_EXPORT extern "C" __attribute__((visibility("default")))

VKB_EXPORT size_t vkblas_b200_q4_bytes(const vkblas_b200_q4_t* w) { return q4_ok(w) ? layout(*w).bytes : 0; }

VKB_EXPORT vkblas_status_t vkblas_b200_q4_pack(const vkblas_b200_q4_t* w, const uint8_t* q, uint32_t ldq,
                                               const void* scales, uint32_t lds, const uint8_t* zeros,
                                               uint32_t ldz, void* packed, void* stream) {
    if (!q4_ok(w) || !q || !packed || !is_al(packed, 256)) return VKBLAS_ERR_PARAM;
    const Layout l = layout(*w);
    if (ldq < (w->K + 1) / 2 || !mat_ok(scales, lds, l.ng) || !w->has_zeros != !zeros || (zeros && ldz < l.ng))
        return VKBLAS_ERR_PARAM;
    OpDevice d;
    if (!op_device(&d)) return VKBLAS_ERR_INIT;
    q4_pack_kernel<<<d.num_sms * 8, 256, 0, static_cast<cudaStream_t>(stream)>>>(
        w->N, w->K, l, q, ldq, static_cast<const uint16_t*>(scales), lds, zeros, ldz, static_cast<uint8_t*>(packed));
    count_launch();
    return op_status(cudaGetLastError());
}

VKB_EXPORT vkblas_status_t vkblas_b200_gemv_q4(const vkblas_b200_q4_t* w, uint32_t M, float alpha,
                                               const void* X, uint32_t ldx, float beta, void* Y,
                                               uint32_t ldy, void* stream) {
    if (!q4_ok(w) || !w->packed || !is_al(w->packed, 256) || M < 1 || M > 16 ||
        !mat_ok(X, ldx, w->K) || !mat_ok(Y, ldy, w->N))
        return VKBLAS_ERR_PARAM;
    OpDevice d;
    if (!op_device(&d)) return VKBLAS_ERR_INIT;
    const Args a{static_cast<const uint8_t*>(w->packed), layout(*w), M, w->N, w->K, w->group,
                 static_cast<const uint16_t*>(X), ldx, Y, ldy, alpha, beta};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return op_status(w->dtype == VKBLAS_DT_F16 ? launch_q4<__half>(a, w->has_zeros != 0, d.num_sms, s)
                                               : launch_q4<__nv_bfloat16>(a, w->has_zeros != 0, d.num_sms, s));
}
