// What the 8-bit block operators' sources share.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace mxq {
// part [n, sets, cols] fp32 summed over n in a fixed order, rounded once to `dtype`: set 0 to out0, set 1 (if there are two)
// to out1; a null output is skipped.
int sum_partials(const float* part, int64_t n, int64_t cols, int sets, void* out0, void* out1, int dtype, cudaStream_t st);
// status word of the 8-bit block products on the current device (0, or MXQ_ERR_DEVICE after a wait gave up)
int fp8_gemm_status(int clear);
// the same of the layer norm's kernels
int norm_status(int clear);
}  // namespace mxq
