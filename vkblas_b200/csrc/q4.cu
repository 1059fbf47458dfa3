// q4.cu -- decode products with 4-bit weights and group scales.
//
//   y[m, n] = alpha * sum_k x[m, k] * s[n, k/G] * (q[n, k] - z[n, k/G]) + beta * y[m, n]
//
// One pass over N K / 2 bytes of weights.  Per group G the products of the
// integers q - z (exact in both 2-byte types) are summed on the tensor cores, and
// that sum times the scale is added to an fp32 sum, so neither the scale nor a
// product is rounded to 2 bytes.
//
// Packed form, written once by vkblas_b200_q4_pack: blocks of 16 weight rows, and in
// a block one record for each step of 128 k, so that a warp's share is one contiguous
// stream.  A record is
//   1024 bytes of weights: lane l = 4 g + t of a warp has 16 bytes of row g, and 512
//     bytes on 16 of row g + 8.  Word w of the 16 holds k = 32 w + 8 t + 0..7, so that a
//     word's MMAs lie in one run of 32 k, whatever multiple of 32 the group is; its nibble
//     i < 4 is k = 2 i and nibble 4 + i is k = 2 i + 1, so that one mask yields a pair of
//     neighbours for the MMA;
//   the scales of the step's 1, 2 or 4 group runs, each [8][2]: rows g and g + 8 side
//     by side, one 32-bit load (a group longer than a step repeats in each: 3 %);
//   the zero points likewise, two nibbles a byte, padded to 16 bytes.
#include <type_traits>

#include "ops.cuh"

namespace vkb {
namespace {

constexpr uint32_t ROWS = 16, STEP = 128, STEP_BYTES = 1024;

// Group runs that a step spans: 1 for groups of a multiple of 128, 2 for other
// multiples of 64, 4 for other multiples of 32.
__host__ __device__ constexpr uint32_t runs_of(uint32_t group) { return group % 128 == 0 ? 1 : group % 64 == 0 ? 2 : 4; }
__host__ __device__ constexpr uint32_t record_bytes(uint32_t runs, bool zeros) {
    return STEP_BYTES + 32 * runs + (zeros ? (runs == 4 ? 32 : 16) : 0);
}

struct Layout {
    uint32_t blocks, steps, ng, runs, rec;
    size_t bytes;
};
Layout layout(const vkblas_b200_q4_t& w) {
    Layout l;
    l.blocks = (w.N - 1) / ROWS + 1;
    l.steps = (w.K - 1) / STEP + 1;
    l.ng = (w.K - 1) / w.group + 1;
    l.runs = runs_of(w.group);
    l.rec = record_bytes(l.runs, w.has_zeros != 0);
    l.bytes = up256((size_t)l.blocks * l.steps * l.rec);
    return l;
}

// One thread per 32-bit word of a record.  Rows past N and k past K are zeros; runs past N or
// the last group have scale 0 (an infinite one would make NaN of the zeros).
__global__ void __launch_bounds__(256) q4_pack_kernel(uint32_t N, uint32_t K, uint32_t group, Layout l, const uint8_t* q,
                                                      uint32_t ldq, const uint16_t* s, uint32_t lds, const uint8_t* z,
                                                      uint32_t ldz, uint32_t* out) {
    const uint32_t per = l.rec / 4;
    const uint64_t words = (uint64_t)l.blocks * l.steps * per, stride = (uint64_t)gridDim.x * 256;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += stride) {
        const uint64_t bs = i / per, n0 = bs / l.steps * ROWS, k0 = bs % l.steps * STEP;
        const uint32_t in = (uint32_t)(i - bs * per);
        uint32_t v = 0;
        if (in < STEP_BYTES / 4) {                               // [half][lane][word]
            const uint32_t w = in & 3, lane = (in >> 2) & 31;
            const uint64_t n = n0 + (lane >> 2) + 8 * (in >> 7), k = k0 + 32 * w + 8 * (lane & 3);
            if (n < N) {
#pragma unroll
                for (uint32_t j = 0; j < 8; j++)
                    if (k + j < K) {
                        const uint32_t nib = (q[n * ldq + (k + j) / 2] >> (4 * (j & 1))) & 15u;
                        v |= nib << (4 * ((j & 1) * 4 + (j >> 1)));
                    }
            }
        } else if (in < STEP_BYTES / 4 + 8 * l.runs) {           // [run][row pair]
            const uint32_t c = in - STEP_BYTES / 4, run = c >> 3;
            const uint64_t n = n0 + (c & 7), g = (k0 + run * (STEP / l.runs)) / group;
            const uint32_t lo = n < N && g < l.ng ? s[n * lds + g] : 0, hi = n + 8 < N && g < l.ng ? s[(n + 8) * lds + g] : 0;
            v = lo | hi << 16;
        } else if (z) {                                          // [run][row pair], a byte each
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const uint32_t c = (in - STEP_BYTES / 4 - 8 * l.runs) * 4 + j, run = c >> 3;
                if (run >= l.runs) break;
                const uint64_t n = n0 + (c & 7), gk = (k0 + run * (STEP / l.runs)) / group, g = gk < l.ng ? gk : l.ng - 1;
                const uint32_t lo = n < N ? z[n * ldz + g] & 15 : 0, hi = n + 8 < N ? z[(n + 8) * ldz + g] & 15 : 0;
                v |= (lo | hi << 4) << (8 * j);
            }
        }
        out[i] = v;
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
    uint32_t M, N, K;
    const uint16_t* x;
    uint32_t ldx;
    void* y;
    uint32_t ldy;
    float alpha, beta;
};

// Packed weights.  Only q4_pack_kernel writes them, an ordinary launch that no kernel of
// launch_pdl overlaps, so they may come by the .nc path; volatile keeps the loads behind
// the wait.  16 bytes as in ld16_stream, scales and zero points through L1.
__device__ __forceinline__ uint4 ldnc_stream(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ldnc_u32(const uint8_t* p) {
    uint32_t v;
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ldnc_u8(const uint8_t* p) {
    uint32_t v;
    asm volatile("ld.global.nc.u8 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

// Eight activations from p, `left` of them inside the row, zeros for the others.  FULL: all
// eight are inside, and p is aligned to AL elements.
template <int AL, bool FULL>
__device__ __forceinline__ uint4 load_x(const uint16_t* p, int32_t left) {
    if constexpr (FULL && AL == 8) {
        return ld16(p);
    } else if constexpr (FULL && AL == 4) {
        const uint2 a = reinterpret_cast<const uint2*>(p)[0], b = reinterpret_cast<const uint2*>(p)[1];
        return make_uint4(a.x, a.y, b.x, b.y);
    } else {
        return gather8(p, left);
    }
}

__device__ __forceinline__ float2 scale_pair(uint32_t v, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ float2 scale_pair(uint32_t v, __nv_bfloat16) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

// This lane's part of one record.
template <bool ZEROS, int RUNS>
struct Rec {
    uint4 lo, hi;
    uint32_t sc[RUNS], zz[RUNS];
    __device__ __forceinline__ void load(const uint8_t* w, const uint8_t* s, const uint8_t* z) {
        lo = ldnc_stream(w);
        hi = ldnc_stream(w + 512);
#pragma unroll
        for (int q = 0; q < RUNS; q++) {
            sc[q] = ldnc_u32(s + 32 * q);
            if (ZEROS) zz[q] = ldnc_u8(z + 8 * q);
        }
    }
};

// One step: sum += scale * ((q - z) x) for each group run.  x is loaded a word's MMAs at a
// time, which holds 4 NT registers of it instead of 16 NT.
template <typename T, int NT, bool ZEROS, int RUNS, typename X>
__device__ __forceinline__ void q4_step(const Rec<ZEROS, RUNS>& r, X&& load, float (&sum)[NT][4]) {
    const uint32_t wl[4] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w}, wh[4] = {r.hi.x, r.hi.y, r.hi.z, r.hi.w};
#pragma unroll
    for (int q = 0; q < RUNS; q++) {
        Dec<T> z0, z1;
        z0.set(ZEROS ? r.zz[q] & 15u : 8u);
        z1.set(ZEROS ? r.zz[q] >> 4 : 8u);
        float d[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) d[n][i] = 0.f;
#pragma unroll
        for (int i = q * (4 / RUNS); i < (q + 1) * (4 / RUNS); i++) {
            uint4 x[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) x[n] = load(i, n);
            uint32_t p0[4], p1[4];
            z0.run(wl[i], p0);
            z1.run(wh[i], p1);
            const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]}, a1[4] = {p0[2], p1[2], p0[3], p1[3]};
#pragma unroll
            for (int n = 0; n < NT; n++) {
                Dec<T>::mma(d[n], a0, x[n].x, x[n].y);
                Dec<T>::mma(d[n], a1, x[n].z, x[n].w);
            }
        }
        const float2 f = scale_pair(r.sc[q], T());
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) sum[n][i] = fmaf(i < 2 ? f.x : f.y, d[n][i], sum[n][i]);
    }
}

// A CTA owns 16 weight rows; its KW warps take contiguous runs of steps and add their
// sums through shared memory in warp order.  Registers are held to what lets 32 warps
// (24 with two token tiles) share an SM: with 7 warps on an SM a step took four times as
// long, since loads, conversion and MMAs of one step depend on each other.
//
// What bounds it (B200, graph replay; 4096 -> 14336 holds 30 MB, 4.7 us of memory time):
// one token 9.4 us, 4 tokens 9.6 us, 16 tokens 17.2 us; 4096 x 4096 3.7 to 3.9 us, of which 2.3
// are the launch.  Before x was loaded a word at a time (10.3 us, one token) a build without the
// arithmetic took 10.2 us and one without the weight loads 10.6 us, so neither memory nor
// arithmetic alone but the short life of a warp (4 to 8 steps between its start and the sum
// with the others) sets the time.  Measured then and dropped: a ring of bulk copies in shared memory for each warp (13.5 us, one token), one
// CTA a SM that keeps x in shared memory and walks over the row blocks (11.9 us; 23 us
// against 16.8 at 13 tokens), and sums of bare nibbles with the zero point taken out at
// the group's end (two thirds of the instructions, 12.1 us).
template <typename T, int NT, bool ZEROS, int RUNS, int AL, int KW>
__global__ void __launch_bounds__(KW * 32, KW == 24 ? 1 : (NT == 2 ? 24 : 32) / KW) q4_gemv_kernel(const Args a) {
    constexpr uint32_t REC = record_bytes(RUNS, ZEROS);
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t b = blockIdx.x, per = (a.l.steps + KW - 1) / KW;
    const uint32_t s0 = min(a.l.steps, warp * per), n = min(a.l.steps, s0 + per) - s0;
    const uint8_t* src = a.w + ((size_t)b * a.l.steps + s0) * REC;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // The warp's whole run into L2 while the kernel ahead may still be at work (a
    // prefetch returns no data, so it need not wait): 3 to 5 % at every size.
    if (lane == 0 && n) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(n * REC) : "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint8_t *wp = src + lane * 16, *sp = src + STEP_BYTES + 4 * g, *zp = src + STEP_BYTES + 32 * RUNS + g;
    // Tokens past M read token 0: a column of the MMA's result that is never stored.
    const uint16_t* xp[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) xp[j] = a.x + (size_t)(g + 8 * j < a.M ? g + 8 * j : 0) * a.ldx + (size_t)s0 * STEP + 8 * t;
    int32_t left = (int32_t)(a.K - s0 * STEP);
    float sum[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) sum[j][i] = 0.f;

    // UN records at once: their loads first, then their arithmetic.  FULL: all their k are inside K.
    auto batch = [&](auto un, auto full) {
        constexpr int UN = decltype(un)::value;
        constexpr bool FULL = decltype(full)::value;
        Rec<ZEROS, RUNS> r[UN];
#pragma unroll
        for (int j = 0; j < UN; j++) r[j].load(wp + j * REC, sp + j * REC, zp + j * REC);
#pragma unroll
        for (int j = 0; j < UN; j++) {
            q4_step<T, NT, ZEROS, RUNS>(r[j], [&](int c, int q) {
                return load_x<AL, FULL>(xp[q] + j * STEP + 32 * c, left - (int32_t)(j * STEP + 32 * c + 8 * t));
            }, sum);
        }
        wp += UN * REC;
        sp += UN * REC;
        zp += UN * REC;
#pragma unroll
        for (int q = 0; q < NT; q++) xp[q] += UN * STEP;
        left -= UN * (int32_t)STEP;
    };
    uint32_t i = 0;
    if constexpr (AL >= 4) {
        // All k of these steps are inside K; a row's last step may be ragged.
        const uint32_t inside = n ? min(n, (uint32_t)left / STEP) : 0u;
        for (; i + 2 <= inside; i += 2) batch(std::integral_constant<int, 2>(), std::true_type());
        if (i < inside) batch(std::integral_constant<int, 1>(), std::true_type()), i++;
        if (i < n) batch(std::integral_constant<int, 1>(), std::false_type());
    } else {
        for (; i + 2 <= n; i += 2) batch(std::integral_constant<int, 2>(), std::false_type());
        if (i < n) batch(std::integral_constant<int, 1>(), std::false_type());
    }

    __shared__ float red[KW][NT * 4][32];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) red[warp][4 * j + i][lane] = sum[j][i];
    __syncthreads();
    // Warp j adds tokens 8 j .. 8 j + 7.  Fragment: (row g, tokens 2t, 2t + 1), (row g + 8, the same).
    if (warp >= NT) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float v = red[0][4 * warp + i][lane];
#pragma unroll
        for (int w = 1; w < KW; w++) v = __fadd_rn(v, red[w][4 * warp + i][lane]);
        const uint32_t row = b * ROWS + g + (i < 2 ? 0 : 8), m = 8 * warp + 2 * t + (i & 1);
        if (row < a.N && m < a.M) {
            T* y = static_cast<T*>(a.y) + (size_t)m * a.ldy + row;
            *y = Elem<T>::from_f(epilogue(a.alpha, v, a.beta, a.beta != 0.f ? Elem<T>::to_f(*y) : 0.f));
        }
    }
}

template <typename T, bool TWO, bool ZEROS, int RUNS>
cudaError_t launch_al(const Args& a, int kw, cudaStream_t s) {
    constexpr int NT = TWO ? 2 : 1;
    const size_t bits = reinterpret_cast<uintptr_t>(a.x) / 2 | (a.M > 1 ? a.ldx : 0);   // in elements
    auto go = [&](auto al) {
        constexpr int AL = decltype(al)::value;
        auto with = [&](auto k) {
            constexpr int KW = decltype(k)::value;
            return launch_pdl(q4_gemv_kernel<T, NT, ZEROS, RUNS, AL, KW>, a.l.blocks, KW * 32, s, a);
        };
        if (kw == 24) return with(std::integral_constant<int, 24>());
        if (kw == 16) return with(std::integral_constant<int, 16>());
        if constexpr (TWO)
            if (kw == 12) return with(std::integral_constant<int, 12>());
        return with(std::integral_constant<int, 8>());
    };
    if (bits % 8 == 0) return go(std::integral_constant<int, 8>());
    if (bits % 4 == 0) return go(std::integral_constant<int, 4>());
    return go(std::integral_constant<int, 1>());
}
template <typename T, bool TWO, bool ZEROS>
cudaError_t launch_runs(const Args& a, int kw, cudaStream_t s) {
    return a.l.runs == 1 ? launch_al<T, TWO, ZEROS, 1>(a, kw, s)
           : a.l.runs == 2 ? launch_al<T, TWO, ZEROS, 2>(a, kw, s) : launch_al<T, TWO, ZEROS, 4>(a, kw, s);
}
// Warps a CTA.  A block's steps are shared by them, so more end sooner, as long as the
// CTAs still run side by side.  Measured (us, with 8 / 12 / 16 / 24 warps):
//   a CTA a SM or fewer       1 token 8192 -> 2048: 7.3 / 6.4 / 5.8 / 4.2
//                             10 tokens 4096 -> 1024: 4.5 / 4.7 / 3.5 / 4.1
//   one token tile, below     14336 -> 4096: 19.9 / 11.5 / 11.4 / 12.2; 4 tokens 8192 -> 5500:
//   24 warps a SM with 8      12.6 / 9.8 / 10.5 / 12.0; above, 4096 -> 14336: 9.3 / 10.8 / 10.8 / 15.2
//   two token tiles (80       16 tokens 4096 x 4096 6.9 / 5.8 / 7.4 / 8.2; 8192 x 8192 20.4 /
//   registers: 24 warps a     17.3 / 19.7 / 21.1; 9 tokens 4096 -> 6000 7.0 / 9.2 / 10.3 /
//   SM, three CTAs of 8 or    11.1; 13 tokens 4100 -> 11003 16.0 / 15.9 / 19.1 / 20.1: waves
//   two of 12)                times steps a warp, with two steps for a CTA's start and end
inline int pick_warps(uint32_t blocks, uint32_t steps, bool two, uint32_t num_sms) {
    if (blocks <= num_sms) return steps >= 48 ? 24 : steps >= 32 ? 16 : 8;
    if (!two) return (uint64_t)blocks * 8 < 24ull * num_sms && steps >= 32 ? 16 : 8;
    auto cost = [&](uint32_t kw) {
        const uint32_t slots = num_sms * (24 / kw);
        return (uint64_t)((blocks - 1) / slots + 1) * ((steps - 1) / kw + 3);
    };
    return cost(12) < cost(8) ? 12 : 8;
}

template <typename T>
cudaError_t launch_q4(const Args& a, bool zeros, int num_sms, cudaStream_t s) {
    const int kw = pick_warps(a.l.blocks, a.l.steps, a.M > 8, (uint32_t)num_sms);
    if (a.M > 8) return zeros ? launch_runs<T, true, true>(a, kw, s) : launch_runs<T, true, false>(a, kw, s);
    return zeros ? launch_runs<T, false, true>(a, kw, s) : launch_runs<T, false, false>(a, kw, s);
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
        w->N, w->K, w->group, l, q, ldq, static_cast<const uint16_t*>(scales), lds, zeros, ldz,
        static_cast<uint32_t*>(packed));
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
    const Args a{static_cast<const uint8_t*>(w->packed), layout(*w), M, w->N, w->K,
                 static_cast<const uint16_t*>(X), ldx, Y, ldy, alpha, beta};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return op_status(w->dtype == VKBLAS_DT_F16 ? launch_q4<__half>(a, w->has_zeros != 0, d.num_sms, s)
                                               : launch_q4<__nv_bfloat16>(a, w->has_zeros != 0, d.num_sms, s));
}
