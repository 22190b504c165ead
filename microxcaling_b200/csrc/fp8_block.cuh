// What the 8-bit block operators' sources share.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace mxq {
// out[c] = sum of part[0..n-1][c] in a fixed order, rounded once to `dtype`
int sum_partials(const float* part, int64_t n, int64_t cols, void* out, int dtype, cudaStream_t st);
// status word of the 8-bit block products on the current device (0, or MXQ_ERR_DEVICE after a wait gave up)
int fp8_gemm_status(int clear);
}  // namespace mxq
