// ops.cu -- data movement shared by the fused language-model products.
#include "ops.cuh"

namespace vkb {
namespace {

// Rows of `cols` 2-byte elements at any alignment -> rows of ldd, a multiple of 8,
// zeros after cols.  A pass over the matrix, bound by memory: a thread gathers
// eight neighbours (lanes read consecutive addresses) and stores 16 bytes.
__global__ void __launch_bounds__(256) copy_rows_kernel(const uint16_t* src, uint32_t ld, uint32_t rows, uint32_t cols,
                                                        uint16_t* dst, uint32_t ldd) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t per = ldd / 8;
    const uint64_t total = (uint64_t)rows * per;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
        const uint32_t r = (uint32_t)(i / per), c = (uint32_t)(i - (uint64_t)r * per) * 8;
        *reinterpret_cast<uint4*>(dst + (size_t)r * ldd + c) = gather8(src + (size_t)r * ld + c, (int64_t)cols - c);
    }
}

}  // namespace

cudaError_t launch_copy_rows(const void* src, uint32_t ld, uint32_t rows, uint32_t cols, void* dst, uint32_t ldd,
                             int num_sms, cudaStream_t s) {
    const uint64_t work = ((uint64_t)rows * (ldd / 8) + 255) / 256, cap = (uint64_t)num_sms * 16;
    return launch_pdl(copy_rows_kernel, (uint32_t)(work < cap ? work : cap), 256, s, static_cast<const uint16_t*>(src), ld,
                      rows, cols, static_cast<uint16_t*>(dst), ldd);
}

}  // namespace vkb
