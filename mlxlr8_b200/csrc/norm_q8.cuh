// Residual add + RMS norm with an E4M3 output and group scales (norm_q8.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace exlr8 {

// group: 32, 64, 128 or hidden.  h_out may be null; residual may be null.
cudaError_t launch_residual_rms_q8(const void* x, const void* residual, const void* w, int act_dtype, int64_t rows,
                                   int hidden, int group, float eps, void* h_out, uint8_t* codes, float* scales,
                                   cudaStream_t s);

}  // namespace exlr8
