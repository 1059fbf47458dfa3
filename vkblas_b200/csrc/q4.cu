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
// follow as [block][group][8][2]: rows g and g + 8 of a block side by side, one
// 32-bit load; zero points likewise, two nibbles a byte.
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
    l.bytes = l.zeros + (w.has_zeros ? up256((size_t)l.blocks * l.ng * (ROWS / 2)) : 0);
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
        const uint64_t bg = i / ROWS, n = bg / l.ng * ROWS + i % ROWS / 2 + 8 * (i & 1), g = bg % l.ng;
        reinterpret_cast<uint16_t*>(out + l.scales)[i] = n < N ? s[n * lds + g] : (uint16_t)0;
        if (z && (i & 1) == 0) {
            const uint32_t z0 = n < N ? z[n * ldz + g] & 15 : 0, z1 = n + 8 < N ? z[(n + 8) * ldz + g] & 15 : 0;
            out[l.zeros + i / 2] = (uint8_t)(z0 | z1 << 4);
        }
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
        const uint32_t v = z * 0x10001u + 0x64006400u;
        lo = *reinterpret_cast<const Pair*>(&v);
        hi = __hfma2(lo, __half2half2(__ushort_as_half((unsigned short)0xBC00u)),      // 960 - lo
                     __half2half2(__ushort_as_half((unsigned short)0x6380u)));
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
        const uint32_t v = z * 0x10001u + 0x43004300u;
        lo = *reinterpret_cast<const Pair*>(&v);
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

// Eight activations from p, `left` of them inside the row, zeros for the others and where
// !ok.  FULL: all eight are inside, and p is aligned to AL elements: predicated vector loads.
template <int AL, bool FULL>
__device__ __forceinline__ uint4 load_x(const uint16_t* p, int32_t left, bool ok) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (FULL && AL == 8) {
        if (ok) v = __ldg(reinterpret_cast<const uint4*>(p));
    } else if constexpr (FULL && AL == 4) {
        if (ok) {
            const uint2 a = __ldg(reinterpret_cast<const uint2*>(p)), b = __ldg(reinterpret_cast<const uint2*>(p) + 1);
            v = make_uint4(a.x, a.y, b.x, b.y);
        }
    } else {
        uint32_t e[8];
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = ok && i < left ? (uint32_t)__ldg(p + i) : 0u;
        v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
    }
    return v;
}

__device__ __forceinline__ float2 scale_pair(uint32_t v, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ float2 scale_pair(uint32_t v, __nv_bfloat16) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

// What a warp carries through its steps.
template <int NT, int RB>
struct Walk {
    const uint8_t* w[RB];            // this lane's 16 bytes of the next step
    const uint32_t* sc[RB];          // the group's scales of rows g and g + 8
    const uint8_t* z[RB];            // and zero points
    const uint16_t* x[NT];           // this lane's first 8 activations of the next step
    bool xok[NT];
    uint32_t in, per;                // runs of 128 / GPS k into the group, and in a group
    uint32_t more;                   // groups after this one
    int32_t left;                    // k from the next step's start to the end of the rows
    float sum[RB][NT][4];
};

// UN steps: all their weights, scales and activations are requested, then used.
template <typename T, int NT, int RB, bool ZEROS, int GPS, int AL, bool FULL, int UN>
__device__ __forceinline__ void q4_steps(Walk<NT, RB>& k, uint32_t t) {
    uint4 w[UN][RB][2], x[UN][4][NT];
    uint32_t sc[UN][RB][GPS], zz[UN][RB][GPS];
#pragma unroll
    for (int j = 0; j < UN; j++)
#pragma unroll
        for (int r = 0; r < RB; r++) {
            w[j][r][0] = ldg_weights(k.w[r] + j * STEP_BYTES);
            w[j][r][1] = ldg_weights(k.w[r] + j * STEP_BYTES + 512);
        }
#pragma unroll
    for (int j = 0; j < UN; j++)
#pragma unroll
        for (int q = 0; q < GPS; q++) {
#pragma unroll
            for (int r = 0; r < RB; r++) {
                sc[j][r][q] = __ldg(k.sc[r]);
                if (ZEROS) zz[j][r][q] = __ldg(k.z[r]);
            }
            // Past K (the end of the last step) the last group stays: x is 0 there.
            if (++k.in == k.per && k.more) {
                k.in = 0;
                k.more--;
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    k.sc[r] += 8;
                    if (ZEROS) k.z[r] += 8;
                }
            }
        }
#pragma unroll
    for (int j = 0; j < UN; j++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int n = 0; n < NT; n++)
                x[j][i][n] = load_x<AL, FULL>(k.x[n] + j * STEP + 32 * i, k.left - j * (int)STEP - 32 * i - 8 * (int)t, k.xok[n]);
#pragma unroll
    for (int j = 0; j < UN; j++)
#pragma unroll
        for (int q = 0; q < GPS; q++) {
            float d[RB][NT][4];
#pragma unroll
            for (int r = 0; r < RB; r++) {
                Dec<T> z0, z1;
                z0.set(ZEROS ? zz[j][r][q] & 15u : 8u);
                z1.set(ZEROS ? zz[j][r][q] >> 4 : 8u);
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++) d[r][n][i] = 0.f;
#pragma unroll
                for (int i = q * (4 / GPS); i < (q + 1) * (4 / GPS); i++) {
                    uint32_t p0[4], p1[4];
                    z0.run(reinterpret_cast<const uint32_t*>(&w[j][r][0])[i], p0);
                    z1.run(reinterpret_cast<const uint32_t*>(&w[j][r][1])[i], p1);
                    const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]}, a1[4] = {p0[2], p1[2], p0[3], p1[3]};
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        Dec<T>::mma(d[r][n], a0, x[j][i][n].x, x[j][i][n].y);
                        Dec<T>::mma(d[r][n], a1, x[j][i][n].z, x[j][i][n].w);
                    }
                }
                const float2 f = scale_pair(sc[j][r][q], T());
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++) k.sum[r][n][i] = fmaf(i < 2 ? f.x : f.y, d[r][n][i], k.sum[r][n][i]);
            }
        }
#pragma unroll
    for (int r = 0; r < RB; r++) k.w[r] += UN * STEP_BYTES;
#pragma unroll
    for (int n = 0; n < NT; n++) k.x[n] += UN * STEP;
    k.left -= UN * (int)STEP;
}

// A CTA owns RB blocks of 16 weight rows; its KW warps take contiguous runs of 128-k
// steps and add their sums through shared memory in warp order.  GPS: groups that a step
// spans (4 for groups of 32 and odd multiples of it, 2 for 64, 1 for multiples of 128).
template <typename T, int NT, int RB, bool ZEROS, int GPS, int AL, int KW>
__global__ void __launch_bounds__(KW * 32, (NT == 2 ? 16 : 32) / KW) q4_gemv_kernel(const Args a) {
    constexpr int UN = 2;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t b0 = blockIdx.x * RB, per = (a.l.steps + KW - 1) / KW;
    uint32_t s = min(a.l.steps, warp * per);
    const uint32_t s1 = min(a.l.steps, s + per);
    Walk<NT, RB> k;
    k.per = a.group / (STEP / GPS);
    const uint32_t run = s * GPS, grp = min(a.l.ng - 1, run / k.per);
    k.in = run - grp * k.per;
    k.more = a.l.ng - 1 - grp;
    k.left = (int32_t)(a.K - s * STEP);
#pragma unroll
    for (int r = 0; r < RB; r++) {
        const size_t b = min(b0 + r, a.l.blocks - 1);        // a block past the last repeats it, unstored
        k.w[r] = a.w + (b * a.l.steps + s) * STEP_BYTES + lane * 16;
        k.sc[r] = reinterpret_cast<const uint32_t*>(a.w + a.l.scales) + (b * a.l.ng + grp) * 8 + g;
        k.z[r] = a.w + a.l.zeros + (b * a.l.ng + grp) * 8 + g;
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
        k.xok[n] = g + 8 * n < a.M;
        k.x[n] = a.x + (size_t)(k.xok[n] ? g + 8 * n : 0) * a.ldx + s * STEP + 8 * t;
    }
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) k.sum[r][n][i] = 0.f;

    if constexpr (AL >= 4) {
        for (; s + UN <= s1 && k.left >= UN * (int)STEP; s += UN) q4_steps<T, NT, RB, ZEROS, GPS, AL, true, UN>(k, t);
        for (; s < s1 && k.left >= (int)STEP; s++) q4_steps<T, NT, RB, ZEROS, GPS, AL, true, 1>(k, t);
    }
    for (; s < s1; s++) q4_steps<T, NT, RB, ZEROS, GPS, AL, false, 1>(k, t);

    __shared__ float red[KW][RB * NT * 4][32];
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) red[warp][4 * (r * NT + n) + i][lane] = k.sum[r][n][i];
    __syncthreads();
    // Warp r NT + n adds block r's tokens 8 n .. 8 n + 7.  Fragment: (row g, tokens 2t, 2t + 1), (row g + 8, the same).
    if (warp >= RB * NT) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float v = red[0][4 * warp + i][lane];
#pragma unroll
        for (int w = 1; w < KW; w++) v = __fadd_rn(v, red[w][4 * warp + i][lane]);
        const uint32_t n = (b0 + warp / NT) * ROWS + g + (i < 2 ? 0 : 8), m = 8 * (warp % NT) + 2 * t + (i & 1);
        if (n < a.N && m < a.M) {
            T* y = static_cast<T*>(a.y) + (size_t)m * a.ldy + n;
            *y = Elem<T>::from_f(epilogue(a.alpha, v, a.beta, a.beta != 0.f ? Elem<T>::to_f(*y) : 0.f));
        }
    }
}

// For more than 8 tokens a warp takes two blocks, which halves the activations' share
// of the L1 traffic (16 tokens' x is 4 KB a step, a block's weights 1 KB).
template <typename T, bool TWO, bool ZEROS, int GPS, int AL>
void launch_kw(const Args& a, int kw, cudaStream_t s) {
    constexpr int NT = TWO ? 2 : 1, RB = 1;
    const uint32_t ctas = (a.l.blocks - 1) / RB + 1;
    if (kw == 4) q4_gemv_kernel<T, NT, RB, ZEROS, GPS, AL, 4><<<ctas, 128, 0, s>>>(a);
    else if (kw == 8) q4_gemv_kernel<T, NT, RB, ZEROS, GPS, AL, 8><<<ctas, 256, 0, s>>>(a);
    else q4_gemv_kernel<T, NT, RB, ZEROS, GPS, AL, 16><<<ctas, 512, 0, s>>>(a);
}
template <typename T, bool TWO, bool ZEROS, int GPS>
void launch_al(const Args& a, int kw, cudaStream_t s) {
    const size_t bits = reinterpret_cast<uintptr_t>(a.x) / 2 | (a.M > 1 ? a.ldx : 0);   // in elements
    if (bits % 8 == 0) launch_kw<T, TWO, ZEROS, GPS, 8>(a, kw, s);
    else if (bits % 4 == 0) launch_kw<T, TWO, ZEROS, GPS, 4>(a, kw, s);
    else launch_kw<T, TWO, ZEROS, GPS, 1>(a, kw, s);
}
template <typename T, bool TWO, bool ZEROS>
void launch_gps(const Args& a, int kw, cudaStream_t s) {
    if (a.group % 128 == 0) launch_al<T, TWO, ZEROS, 1>(a, kw, s);
    else if (a.group % 64 == 0) launch_al<T, TWO, ZEROS, 2>(a, kw, s);
    else launch_al<T, TWO, ZEROS, 4>(a, kw, s);
}
template <typename T>
cudaError_t launch_q4(const Args& a, bool zeros, int num_sms, cudaStream_t s) {
    const bool two = a.M > 8;
    // Warps a CTA: enough that all SMs together hold about 24 warps each, but not more
    // than one a step of 128 k.
    const uint64_t ctas = a.l.blocks;
    int kw = 4;
    while (kw < 16 && ctas * kw < 24ull * num_sms && a.l.steps >= 2u * kw) kw *= 2;
    if (two) zeros ? launch_gps<T, true, true>(a, kw, s) : launch_gps<T, true, false>(a, kw, s);
    else zeros ? launch_gps<T, false, true>(a, kw, s) : launch_gps<T, false, false>(a, kw, s);
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
