// row_copy.hip -- factor matrices between host rows of k floats and device rows of ld >= k floats (the
// models' set and get calls).
//
// One linear copy where ld == k.  Else the rows go through a packed device buffer in pieces, a kernel
// beside each copy: a strided copy of pageable host memory takes 13 us a row here (1 M rows of 512 bytes:
// 6.8 s, against 0.05 s in one piece).
#include <algorithm>

#include "mml_internal.h"

namespace {

constexpr int64_t kPiece = (int64_t)16 << 20;  // floats of the packed buffer at most

__global__ __launch_bounds__(256) void pack_rows_kernel(float* __restrict__ dst,
                                                        const float* __restrict__ src, int64_t rows,
                                                        int32_t k, int64_t ld) {
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < rows * k;
         x += (int64_t)gridDim.x * 256)
        dst[x] = src[x / k * ld + x % k];
}
// the columns from k on become 0
__global__ __launch_bounds__(256) void unpack_rows_kernel(float* __restrict__ dst,
                                                          const float* __restrict__ src, int64_t rows,
                                                          int32_t k, int32_t ld) {
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < rows * ld;
         x += (int64_t)gridDim.x * 256) {
        const int64_t r = x / ld;
        const int32_t f = (int32_t)(x - r * ld);
        dst[x] = f < k ? src[r * k + f] : 0.0f;
    }
}
uint32_t grid_of(int64_t n) { return (uint32_t)std::min<int64_t>((n + 255) / 256, 8192); }

}  // namespace

namespace mml {

void upload_rows(hipStream_t st, float* dst, int32_t ld, const float* src, int32_t k, int64_t rows) {
    if (rows == 0) return;
    if (ld == k) {
        MML_HIP(hipMemcpyAsync(dst, src, sizeof(float) * rows * k, hipMemcpyHostToDevice, st));
        return;
    }
    const int64_t piece = std::min(rows, std::max<int64_t>(1, kPiece / k));
    DeviceArray<float> packed;
    packed.alloc((size_t)piece * k);
    for (int64_t r = 0; r < rows; r += piece) {
        const int64_t n = std::min(piece, rows - r);
        MML_HIP(hipMemcpyAsync(packed.get(), src + r * k, sizeof(float) * n * k,
                               hipMemcpyHostToDevice, st));
        unpack_rows_kernel<<<grid_of(n * ld), 256, 0, st>>>(dst + r * ld, packed.get(), n, k, ld);
        MML_HIP(hipGetLastError());
    }
    MML_HIP(hipStreamSynchronize(st));  // the packed buffer is done with
}

void download_rows(hipStream_t st, float* dst, int32_t k, const float* src, int32_t ld, int64_t rows) {
    if (rows == 0) return;
    if (ld == k) {
        MML_HIP(hipMemcpyAsync(dst, src, sizeof(float) * rows * k, hipMemcpyDeviceToHost, st));
        return;
    }
    const int64_t piece = std::min(rows, std::max<int64_t>(1, kPiece / k));
    DeviceArray<float> packed;
    packed.alloc((size_t)piece * k);
    for (int64_t r = 0; r < rows; r += piece) {
        const int64_t n = std::min(piece, rows - r);
        pack_rows_kernel<<<grid_of(n * k), 256, 0, st>>>(packed.get(), src + r * ld, n, k, ld);
        MML_HIP(hipGetLastError());
        MML_HIP(hipMemcpyAsync(dst + r * k, packed.get(), sizeof(float) * n * k,
                               hipMemcpyDeviceToHost, st));
    }
    MML_HIP(hipStreamSynchronize(st));
}

}  // namespace mml
