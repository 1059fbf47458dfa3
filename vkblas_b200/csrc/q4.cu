// q4.cu -- decode products with 4-bit weights and group scales.
//
//   y[m, n] = alpha * sum_k x[m, k] * s[n, k/G] * (q[n, k] - z[n, k/G]) + beta * y[m, n]
#include "ops.cuh"

namespace vkb {
namespace {

// Packed form: [N][K/2 rounded up to 4 bytes of words][scales N x ng][zeros N x ng].
struct Layout {
    uint32_t ng;
    size_t row_bytes, scales, zeros, bytes;
};
Layout layout(const vkblas_b200_q4_t& w) {
    Layout l;
    l.ng = (w.K - 1) / w.group + 1;
    l.row_bytes = ((size_t)w.K + 1) / 2;
    l.scales = up256(l.row_bytes * w.N);
    l.zeros = l.scales + up256((size_t)w.N * l.ng * 2);
    l.bytes = l.zeros + (w.has_zeros ? up256((size_t)w.N * l.ng) : 0);
    return l;
}

__global__ void q4_pack_kernel(uint32_t N, Layout l, const uint8_t* q, uint32_t ldq, const uint16_t* s,
                               uint32_t lds, const uint8_t* z, uint32_t ldz, uint8_t* out) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < l.row_bytes * N; i += (uint64_t)gridDim.x * 256)
        out[i] = q[i / l.row_bytes * ldq + i % l.row_bytes];
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < (uint64_t)N * l.ng; i += (uint64_t)gridDim.x * 256) {
        reinterpret_cast<uint16_t*>(out + l.scales)[i] = s[i / l.ng * lds + i % l.ng];
        if (z) out[l.zeros + i] = z[i / l.ng * ldz + i % l.ng] & 15;
    }
}

template <typename T>
__global__ void q4_gemv_kernel(Layout l, const uint8_t* w, uint32_t K, uint32_t group, bool has_zeros,
                               uint32_t M, uint32_t N, float alpha, const T* X, uint32_t ldx, float beta,
                               T* Y, uint32_t ldy) {
    const uint32_t n = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
    if (n >= N) return;
    for (uint32_t m = 0; m < M; m++) {
        float sum = 0.f;
        for (uint32_t k = lane; k < K; k += 32) {
            const size_t g = (size_t)n * l.ng + k / group;
            const int q = w[n * l.row_bytes + k / 2] >> (4 * (k & 1)) & 15;
            const int z = has_zeros ? w[l.zeros + g] : 8;
            const float s = Elem<T>::to_f(reinterpret_cast<const T*>(w + l.scales)[g]);
            sum = fmaf(Elem<T>::to_f(X[(size_t)m * ldx + k]), s * (q - z), sum);
        }
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (lane == 0) {
            T* y = Y + (size_t)m * ldy + n;
            *y = Elem<T>::from_f(epilogue(alpha, sum, beta, beta != 0.f ? Elem<T>::to_f(*y) : 0.f));
        }
    }
}

bool q4_ok(const vkblas_b200_q4_t* w) {
    return w && two_byte(w->dtype) && w->N && w->K && w->group && w->group % 32 == 0;
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
    if (ldq < l.row_bytes || !mat_ok(scales, lds, l.ng) || !w->has_zeros != !zeros ||
        (zeros && ldz < l.ng))
        return VKBLAS_ERR_PARAM;
    OpDevice d;
    if (!op_device(&d)) return VKBLAS_ERR_INIT;
    q4_pack_kernel<<<d.num_sms * 8, 256, 0, static_cast<cudaStream_t>(stream)>>>(
        w->N, l, q, ldq, static_cast<const uint16_t*>(scales), lds, zeros, ldz, static_cast<uint8_t*>(packed));
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
    const Layout l = layout(*w);
    const uint8_t* p = static_cast<const uint8_t*>(w->packed);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint32_t blocks = (w->N - 1) / 8 + 1;
    if (w->dtype == VKBLAS_DT_F16)
        q4_gemv_kernel<__half><<<blocks, 256, 0, s>>>(l, p, w->K, w->group, w->has_zeros != 0, M, w->N, alpha,
            static_cast<const __half*>(X), ldx, beta, static_cast<__half*>(Y), ldy);
    else
        q4_gemv_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>(l, p, w->K, w->group, w->has_zeros != 0, M, w->N, alpha,
            static_cast<const __nv_bfloat16*>(X), ldx, beta, static_cast<__nv_bfloat16*>(Y), ldy);
    count_launch();
    return op_status(cudaGetLastError());
}
