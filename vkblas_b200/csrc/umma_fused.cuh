// umma_fused.cuh -- tcgen05 products whose results are used in the epilogue:
// the gated block (gated.cu) and the cross entropy of a linear head (xent.cu).
//
// The main loop is the 2-byte GEMM's of umma_gemm.cu: A (M x K) and B (N x K)
// K-major through TMA into a shared-memory ring, 256-row tiles on 2-CTA
// clusters (PAIR) or 128-row tiles on single CTAs, 256 columns of B per tile, two
// TMEM accumulators, one issuing thread.  Here B's 256 rows may come from two
// matrices (128 each), and the epilogue has eight warps: two share a TMEM lane
// quarter, so a thread holds one row and half of the tile's columns.  What they
// do with the accumulator is the policy EPI's:
//   SEG_KB    k-blocks accumulated in one TMEM buffer before the epilogue adds
//             them to fp32 sums in registers; 0: the whole of K.  The tensor
//             core's accumulation truncates, the epilogue's adds round to nearest
//             (bf16 logits of 8 and more, K = 4096: 4.2e-6 of them too small in one
//             sum, 4.8e-7 in segments of 512).
//   TWO_B     gate and up rows: the first half of a tile's columns are rows of the first
//             matrix, the second half the same rows of the second.
//   run()     the epilogue of one tile.
// No TMA load uses cluster multicast; every wait is bounded (umma.cuh).
#pragma once
#include <atomic>
#include <cstring>

#include "ops.cuh"
#include "umma.cuh"

namespace vkb {
namespace fused {

using namespace umma;

constexpr uint32_t BM = 128, BN = 256, BK = 64;          // 64 2-byte k: one 128-byte swizzle row
constexpr uint32_t A_BYTES = BM * 128;
constexpr uint32_t EPI_WARPS = 8, EPI_WARP0 = 4;
constexpr uint32_t THREADS = 32 * (EPI_WARP0 + EPI_WARPS);
constexpr uint32_t BOX_BYTES = 32 * 128;                 // 32 rows x 64 2-byte columns
constexpr uint64_t WAIT_LIMIT_NS = 2000000000ull, DRAIN_LIMIT_NS = 200000000ull;
// Register split of the segmented epilogue (128 fp32 sums a thread): warps 0-3 drop
// to REGS_LOW, the eight epilogue warps rise to REGS_HIGH.
constexpr uint32_t REGS_LOW = 56, REGS_HIGH = 208;

struct __align__(64) Params {
    CUtensorMap tmA, tmB[2];
    uint32_t M, N, K;                   // N: rows of each B matrix
    uint32_t half;                      // half of a tile's columns (pick_half)
    uint32_t tiles_m, tiles_n, num_kb, total, group_m;
    int* status;
};

template <bool PAIR>
struct Ring {
    // Pairs: each CTA holds 128 rows of A and half of B; three stages of two
    // k-blocks (64 KB), one wait and one commit per eight MMAs.  Single CTAs: four
    // stages of one k-block (48 KB).
    static constexpr uint32_t KBS = PAIR ? 2 : 1, STAGES = PAIR ? 3 : 4;
    static constexpr uint32_t B_ROWS = PAIR ? BN / 2 : BN;
    static constexpr uint32_t KB_BYTES = A_BYTES + B_ROWS * 128;
    static constexpr uint32_t STAGE_BYTES = KBS * KB_BYTES;
    static constexpr uint32_t BM_TILE = PAIR ? 2 * BM : BM;
    static constexpr uint32_t SMEM = STAGES * STAGE_BYTES + EPI_WARPS * BOX_BYTES + 1024 + 256;
};

// What a policy's run() gets for a tile.
struct Tile {
    uint32_t m0, m;              // first row of this warp's 32, this thread's row
    uint32_t nb;                 // column block
    uint32_t half;               // which half of the columns this warp has (0 or 1)
    uint32_t tmem;               // TMEM address of this warp's lanes, column 0 of the buffer
    uint32_t box;                // this warp's staging box
    int lane;
};

__device__ __forceinline__ void tile_of(const Params& p, uint32_t u, uint32_t& mb, uint32_t& nb) {
    const uint32_t per = p.group_m * p.tiles_n, group = u / per, first = group * p.group_m;
    const uint32_t rows = min(p.tiles_m - first, p.group_m), in = u - group * per;
    mb = first + in % rows;
    nb = in / rows;
}

// A row-major 2-byte output.  vec: rows start on 16 bytes, 16-byte units apart.
struct Out {
    void* p;
    uint32_t ld, rows, cols, vec;
};
inline Out output(void* p, uint32_t ld, uint32_t rows, uint32_t cols) {
    return {p, ld, rows, cols, is_al(p, 16) && ld % 8 == 0 ? 1u : 0u};
}

// Stores `width` (at most 64) columns, n0 onwards, of this warp's 32 rows: each thread
// brings its row as 32 packed pairs, the warp's box in shared memory turns them into
// whole 128-byte pieces of rows (16-byte unit g of row r sits at g ^ (r % 8): no bank
// conflicts either way), and eight lanes store a row's 64 columns together.  Where rows do
// not start on 16 bytes the warp goes row by row, its 2- or 4-byte stores neighbours
// (1150 x 11223, three outputs, K = 256: 159 us with eight 2-byte stores a lane and unit
// instead, 66 us so, 35 us with aligned rows).
__device__ __forceinline__ void store_rows(const Out& o, const Tile& t, uint32_t n0, uint32_t width,
                                           const uint32_t (&v)[32]) {
    if (n0 >= o.cols || t.m0 >= o.rows) return;          // warp-uniform
    const uint32_t nc = min(width, o.cols - n0), nr = min(32u, o.rows - t.m0);
    __syncwarp();
#pragma unroll
    for (uint32_t g = 0; g < 8; g++)
        st_shared_v4(t.box + (uint32_t)t.lane * 128u + ((g ^ ((uint32_t)t.lane & 7u)) << 4),
                     make_uint4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]));
    __syncwarp();
    uint16_t* out = static_cast<uint16_t*>(o.p) + (size_t)t.m0 * o.ld + n0;
    const uint32_t lane = (uint32_t)t.lane;
    if (o.vec && nc % 8u == 0) {
        const uint32_t g = lane & 7u;
        if (g * 8u >= nc) return;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const uint32_t r = 4u * i + (lane >> 3);
            if (r >= nr) break;
            uint4 w;
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                         : "r"(t.box + r * 128u + ((g ^ (r & 7u)) << 4)) : "memory");
            *reinterpret_cast<uint4*>(out + (size_t)r * o.ld + g * 8u) = w;
        }
        return;
    }
#pragma unroll 4
    for (uint32_t r = 0; r < nr; r++) {
        uint16_t* q = out + (size_t)r * o.ld;
        auto unit = [&](uint32_t c) { return t.box + r * 128u + (((c >> 3) ^ (r & 7u)) << 4) + (c & 7u) * 2u; };
        if ((reinterpret_cast<uintptr_t>(q) & 3u) == 0) {
            const uint32_t c = 2u * lane;
            uint32_t w;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(unit(c)) : "memory");
            if (c + 1 < nc) *reinterpret_cast<uint32_t*>(q + c) = w;
            else if (c < nc) q[c] = (uint16_t)w;
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 2; j++) {
                const uint32_t c = lane + 32u * j;
                uint16_t w;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(unit(c)) : "memory");
                if (c < nc) q[c] = w;
            }
        }
    }
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool BF16, typename EPI, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1)
    fused_kernel(const __grid_constant__ Params p, const __grid_constant__ typename EPI::Args ea) {
    using R = Ring<PAIR>;
    constexpr uint32_t STAGES = R::STAGES, KBS = R::KBS, NBUF = 2;
    constexpr uint32_t SEG = EPI::SEG_KB;
    static_assert(SEG % KBS == 0, "a segment is whole stages");
    const uint32_t idesc = instr_desc(BF16 ? 1u : 0u, false, false, R::BM_TILE, 2u * p.half);
    const uint32_t kb_bytes = A_BYTES + (PAIR ? 1u : 2u) * p.half * 128u;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), padb = (1024u - (raw & 1023u)) & 1023u;
    const uint32_t sbase = raw + padb;
    const uint32_t boxes = sbase + STAGES * R::STAGE_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem_raw + padb + STAGES * R::STAGE_BYTES + EPI_WARPS * BOX_BYTES);
    const uint32_t bar0 = smem_u32(bars);
    auto full_bar = [&](uint32_t s) { return bar0 + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar0 + 8u * (STAGES + s); };
    auto tfull_bar = [&](uint32_t a) { return bar0 + 8u * (2 * STAGES + a); };
    auto tempty_bar = [&](uint32_t a) { return bar0 + 8u * (2 * STAGES + NBUF + a); };
    const uint32_t drain_bar = bar0 + 8u * (2 * STAGES + 2 * NBUF);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 2 * NBUF + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const uint32_t warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
    const bool issuer = rank == 0;
    const uint32_t unit0 = PAIR ? blockIdx.x >> 1 : blockIdx.x;
    const uint32_t ustride = PAIR ? gridDim.x >> 1 : gridDim.x;
    auto to_issuer = [&](uint32_t bar) { return PAIR ? mapa_shared(bar, 0) : bar; };

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < STAGES; s++) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (uint32_t a = 0; a < NBUF; a++) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), (PAIR ? 2u : 1u) * 32u * EPI_WARPS);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
        fence_proxy_async_smem();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&p.tmA);
        prefetch_tmap(&p.tmB[0]);
        if (EPI::TWO_B) prefetch_tmap(&p.tmB[1]);
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            tmem_alloc_pair(smem_u32(tmem_slot), NBUF * BN);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(tmem_slot), NBUF * BN);
            tmem_relinquish();
        }
    }
    __syncthreads();
    if constexpr (PAIR) cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp < EPI_WARP0) {
        if constexpr (SEG != 0) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_LOW));
        if (warp == 0 && lane == 0) {
            // ---------------------------------------------------------- producer
            // Launched as a programmatic dependent: nothing is read before the
            // kernels ahead on the stream are done.
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            uint32_t stage = 0, phase = 0, issued = 0, parity = 0;
            bool ok = true;
            for (uint32_t u = unit0; ok && u < p.total; u += ustride) {
                uint32_t mb, nb;
                tile_of(p, u, mb, nb);
                const int32_t m0 = (int32_t)(mb * R::BM_TILE + rank * BM);
                for (uint32_t kb = 0; kb < p.num_kb; kb += KBS) {
                    const uint32_t nk = min(KBS, p.num_kb - kb);
                    if (!wait_bar(empty_bar(stage), phase ^ 1u, abort_flag, p.status, DS_TIMEOUT_PRODUCER,
                                  WAIT_LIMIT_NS)) {
                        ok = false;
                        break;
                    }
                    const uint32_t fb = to_issuer(full_bar(stage));
                    if (issuer) mbar_arrive_expect_tx(full_bar(stage), (PAIR ? 2u : 1u) * nk * kb_bytes);
                    auto load = [&](uint32_t dst, const CUtensorMap* m, int32_t k0, int32_t r0) {
                        if constexpr (PAIR) tma_load_3d_pair(dst, m, fb, k0, r0, 0);
                        else tma_load_3d(dst, m, fb, k0, r0, 0);
                    };
                    for (uint32_t i = 0; i < nk; i++) {
                        const uint32_t sA = sbase + stage * R::STAGE_BYTES + i * R::KB_BYTES;
                        const int32_t k0 = (int32_t)((kb + i) * BK);
                        load(sA, &p.tmA, k0, m0);
                        // B in boxes of `half` rows: this CTA's half of a pair tile, or both.
#pragma unroll
                        for (uint32_t j = 0; j < (PAIR ? 1u : 2u); j++) {
                            const uint32_t h = PAIR ? rank : j;
                            if constexpr (EPI::TWO_B)
                                load(sA + A_BYTES + j * p.half * 128u, &p.tmB[h], k0, (int32_t)(nb * p.half));
                            else
                                load(sA + A_BYTES + j * p.half * 128u, &p.tmB[0], k0, (int32_t)((2u * nb + h) * p.half));
                        }
                    }
                    issued |= 1u << stage;
                    parity = (parity & ~(1u << stage)) | (phase << stage);
                    if (++stage == STAGES) stage = 0, phase ^= 1u;
                }
            }
            // Never leave with copies in flight (as in umma_gemm.cu).
            for (uint32_t s = 0; s < STAGES; s++)
                if (issued & (1u << s))
                    drain_bar_wait(issuer ? full_bar(s) : empty_bar(s), (parity >> s) & 1u, p.status,
                                   DS_TIMEOUT_PRODUCER, DRAIN_LIMIT_NS);
        } else if (warp == 1 && lane == 0 && issuer) {
            // ---------------------------------------------------------- MMA issuer
            uint32_t stage = 0, phase = 0, u = 0;
            bool ok = true;
            for (uint32_t w = unit0; ok && w < p.total; w += ustride) {
                const uint32_t seg = SEG ? SEG : p.num_kb;
                for (uint32_t kb0 = 0; ok && kb0 < p.num_kb; kb0 += seg, u++) {
                    const uint32_t buf = u % NBUF, kb1 = min(p.num_kb, kb0 + seg);
                    if (!wait_bar(tempty_bar(buf), ((u / NBUF) & 1u) ^ 1u, abort_flag, p.status, DS_TIMEOUT_MMA,
                                  WAIT_LIMIT_NS)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d = tmem_base + buf * BN;
                    for (uint32_t kb = kb0; kb < kb1; kb += KBS) {
                        const uint32_t nk = min(KBS, kb1 - kb);
                        if (!wait_bar(full_bar(stage), phase, abort_flag, p.status, DS_TIMEOUT_MMA, WAIT_LIMIT_NS)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t sA = sbase + stage * R::STAGE_BYTES;
                        const uint64_t ad0 = smem_desc_sw128(sA, 16, 1024);
                        const uint64_t bd0 = smem_desc_sw128(sA + A_BYTES, 16, 1024);
#pragma unroll
                        for (uint32_t i = 0; i < KBS; i++) {
                            if (i >= nk) break;
#pragma unroll
                            for (uint32_t j = 0; j < 4; j++) {
                                const uint64_t off = ((i * R::KB_BYTES) >> 4) + j * 2u;
                                const uint32_t acc = (kb == kb0 && i == 0 && j == 0) ? 0u : 1u;
                                if constexpr (PAIR) mma_f16_pair(d, ad0 + off, bd0 + off, idesc, acc);
                                else mma_f16(d, ad0 + off, bd0 + off, idesc, acc);
                            }
                        }
                        if constexpr (PAIR) tc_commit_pair_mc(empty_bar(stage), 0x3);
                        else tc_commit(empty_bar(stage));
                        if (++stage == STAGES) stage = 0, phase ^= 1u;
                    }
                    if (!ok) break;
                    if constexpr (PAIR) tc_commit_pair_mc(tfull_bar(buf), 0x3);
                    else tc_commit(tfull_bar(buf));
                }
            }
            if constexpr (PAIR) tc_commit_pair(drain_bar);
            else tc_commit(drain_bar);
            drain_bar_wait(drain_bar, 0, p.status, DS_TIMEOUT_MMA, DRAIN_LIMIT_NS);
        }
    } else {
        if constexpr (SEG != 0) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_HIGH));
        // -------------------------------------------------------------- epilogue
        asm volatile("griddepcontrol.wait;" ::: "memory");
        const uint32_t q = warp & 3u;
        Tile t;
        t.half = (warp - EPI_WARP0) / 4u;
        t.box = boxes + (warp - EPI_WARP0) * BOX_BYTES;
        t.lane = lane;
        uint32_t u = 0;
        bool ok = true;
        // The next accumulator of this tile: false when the CTA aborts.
        auto acquire = [&]() {
            const uint32_t buf = u % NBUF;
            ok = wait_bar(tfull_bar(buf), (u / NBUF) & 1u, abort_flag, p.status, DS_TIMEOUT_EPILOGUE, WAIT_LIMIT_NS);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            t.tmem = tmem_base + ((q * 32u) << 16) + buf * BN;
            return ok;
        };
        auto release = [&]() {
            tc_fence_before();
            if constexpr (PAIR) mbar_arrive_cluster(to_issuer(tempty_bar(u % NBUF)));
            else mbar_arrive(tempty_bar(u % NBUF));
            u++;
        };
        for (uint32_t w = unit0; ok && w < p.total; w += ustride) {
            uint32_t mb;
            tile_of(p, w, mb, t.nb);
            t.m0 = mb * R::BM_TILE + rank * BM + q * 32u;
            t.m = t.m0 + (uint32_t)lane;
            EPI::run(p, ea, t, acquire, release);
        }
    }
    __syncthreads();
    if constexpr (PAIR) cluster_sync();      // a pair leaves together
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR) tmem_dealloc_pair(tmem_base, NBUF * BN);
        else tmem_dealloc(tmem_base, NBUF * BN);
    }
}

// ---------------------------------------------------------------------- host
struct Matrix {
    const void* p;
    uint32_t ld;
};

// Half of a tile's columns: 128, and less (a multiple of 32, at least 32) where tiles
// would not reach every worker, so that more of them do.  With several waves of tiles
// narrower ones do not pay: a k-block costs 0.379 us with 256 columns and 0.343 with 208
// (4096 tokens, 4096 -> 14336), since the A operand's share of the feed stays.
inline uint32_t pick_half(uint32_t M, uint32_t N, bool two_b, int num_sms) {
    const bool pair = M >= 2 * BM;
    const uint64_t tiles_m = (M - 1) / (pair ? 2 * BM : BM) + 1, workers = (uint32_t)num_sms / (pair ? 2 : 1);
    for (uint32_t h = 32; h < 128; h += 32)
        if (tiles_m * ((N - 1) / (two_b ? h : 2 * h) + 1) <= workers) return h;
    return 128;
}

// Launches the kernel over the tiles of an M x N problem (N rows in each B
// matrix): 256-row pair tiles when M fills them, else 128-row tiles.
template <bool BF16, typename EPI, bool PAIR>
cudaError_t launch(Params& p, const Matrix& a, const Matrix (&b)[2], const typename EPI::Args& ea, int num_sms,
                   cudaStream_t s) {
    using R = Ring<PAIR>;
    auto kern = fused_kernel<BF16, EPI, PAIR>;
    static std::atomic<uint64_t> ready{0};           // one bit per device
    static int clusters[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    cudaLaunchConfig_t c = {};
    cudaLaunchAttribute at[2];
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = R::SMEM;
    c.attrs = at;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    if (!(ready.load() & bit)) {
        cudaFuncAttributes fa;
        cudaError_t e = cudaFuncGetAttributes(&fa, kern);
        if (e != cudaSuccess) return e;
        // The register split has to fit what the block is launched with: an
        // unsatisfiable setmaxnreg.inc would wait for good.
        if (EPI::SEG_KB != 0 && (uint64_t)(fa.numRegs & ~7) * THREADS <
                                    128ull * REGS_LOW + (THREADS - 128ull) * REGS_HIGH)
            return cudaErrorNotSupported;
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)R::SMEM);
        if (e != cudaSuccess) return e;
        if (PAIR) {
            c.gridDim = dim3((uint32_t)num_sms & ~1u);
            c.numAttrs = 1;
            int n = 0;
            e = cudaOccupancyMaxActiveClusters(&n, kern, &c);
            if (e != cudaSuccess) return e;
            if (n < 1) return cudaErrorNotSupported;
            clusters[dev & 63] = n;
        }
        ready.fetch_or(bit);
    }
    const uint32_t wide = PAIR ? (uint32_t)clusters[dev & 63] : (uint32_t)num_sms;
    p.tiles_m = (p.M - 1) / R::BM_TILE + 1;
    p.tiles_n = (p.N - 1) / (EPI::TWO_B ? p.half : 2 * p.half) + 1;
    p.num_kb = (p.K - 1) / BK + 1;
    p.group_m = p.tiles_m <= 16 ? 16 : 8;            // as measured for the GEMM (umma_gemm.cu)
    const uint64_t total = (uint64_t)p.tiles_m * p.tiles_n;
    if (total >= (1ull << 31)) return cudaErrorInvalidConfiguration;
    p.total = (uint32_t)total;
    // K-major operands in boxes of 64 k: 128 rows of A, and of B half a tile's.
    if (!encode_tmap_sw128(&p.tmA, BF16, a.p, p.K, p.M, a.ld, BK, BM)) return cudaErrorNotSupported;
    for (int i = 0; i < (EPI::TWO_B ? 2 : 1); i++)
        if (!encode_tmap_sw128(&p.tmB[i], BF16, b[i].p, p.K, p.N, b[i].ld, BK, p.half))
            return cudaErrorNotSupported;
    c.gridDim = dim3((PAIR ? 2u : 1u) * (p.total < wide ? p.total : wide));
    c.stream = s;
    unsigned n = PAIR ? 1 : 0;
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    c.numAttrs = n + 1;
    const cudaError_t e = cudaLaunchKernelEx(&c, kern, p, ea);
    count_launch();
    return e;
}

template <bool BF16, typename EPI>
cudaError_t launch_any(uint32_t M, uint32_t N, uint32_t K, uint32_t half, const Matrix& a, const Matrix (&b)[2],
                       const typename EPI::Args& ea, const OpDevice& d, cudaStream_t s) {
    Params p;
    memset(&p, 0, sizeof(p));
    p.M = M, p.N = N, p.K = K, p.half = half;
    p.status = d.status;
    return M >= 2 * BM ? launch<BF16, EPI, true>(p, a, b, ea, d.num_sms, s)
                       : launch<BF16, EPI, false>(p, a, b, ea, d.num_sms, s);
}

}  // namespace fused

// Operands that TMA cannot read (rows not whole 16-byte units apart, or a start off
// the 16-byte grid) are copied into the workspace once, in rows of a multiple of 8.
inline bool tma_readable(const void* p, uint32_t ld) { return is_al(p, 16) && ld % 8 == 0; }
struct Operand2 {
    const void* p;
    uint32_t ld;
    bool copied;
    void* copy;
};
// The operand as the kernels will see it, with room for its copy taken if needed.
inline Operand2 operand(Carver& c, const void* p, uint32_t ld, uint32_t rows, uint32_t cols) {
    if (tma_readable(p, ld)) return {p, ld, false, nullptr};
    const uint32_t l = up8(cols);
    void* copy = c.take<uint16_t>((size_t)rows * l);
    return {copy, l, true, copy};
}
inline cudaError_t fill(const Operand2& o, const void* p, uint32_t ld, uint32_t rows, uint32_t cols, int num_sms,
                        cudaStream_t s) {
    return o.copied ? launch_copy_rows(p, ld, rows, cols, o.copy, o.ld, num_sms, s) : cudaSuccess;
}

}  // namespace vkb
