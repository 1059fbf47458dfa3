// simple.cuh -- a plain tiled product with fp32 sums for any layout: operands
// come through functors a(m, k) and b(n, k), results go to one, so every
// product of the fused operators is an instance of it.  64 x 64 outputs per
// 256-thread block, 4 x 4 per thread, k in order; NB products share A.
#pragma once
#include "common.cuh"

namespace vkb {

template <int NB, typename FA, typename FB, typename FE>
__global__ void __launch_bounds__(256) simple_product(uint32_t M, uint32_t N, uint32_t K, FA a, FB b,
                                                      FE epi) {
    __shared__ float As[16][65], Bs[NB][16][65];
    const uint32_t n0 = blockIdx.x * 64u, m0 = blockIdx.y * 64u;
    const uint32_t tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[NB][4][4] = {};
    for (uint32_t k0 = 0; k0 < K; k0 += 16) {
        for (uint32_t e = threadIdx.x; e < 64 * 16; e += 256) {
            const uint32_t r = e >> 4, c = e & 15, k = k0 + c;
            As[c][r] = (m0 + r < M && k < K) ? a(m0 + r, k) : 0.f;
#pragma unroll
            for (int i = 0; i < NB; i++) Bs[i][c][r] = (n0 + r < N && k < K) ? b(i, n0 + r, k) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < 16; kk++)
#pragma unroll
            for (int q = 0; q < NB; q++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        acc[q][i][j] = fmaf(As[kk][ty * 4 + i], Bs[q][kk][tx * 4 + j], acc[q][i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            float v[NB];
#pragma unroll
            for (int q = 0; q < NB; q++) v[q] = acc[q][i][j];
            if (m < M && n < N) epi(m, n, v);
        }
}

template <int NB, typename FA, typename FB, typename FE>
cudaError_t launch_simple(uint32_t M, uint32_t N, uint32_t K, FA a, FB b, FE e, cudaStream_t s) {
    if ((M + 63) / 64 > 65535u) return cudaErrorInvalidConfiguration;
    simple_product<NB><<<dim3((N + 63) / 64, (M + 63) / 64), 256, 0, s>>>(M, N, K, a, b, e);
    count_launch();
    return cudaGetLastError();
}

}  // namespace vkb
