// Linear layers with 4-bit affine weights and group scales (affine4.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace exlr8 {

struct Affine4Args {
  const void* x;          // [rows][in] activations, or E4M3 codes
  int x_dtype;            // EXLR8_DTYPE_*
  const float* x_scales;  // [rows][in / x_group] of E4M3 codes, else null
  int x_group;
  int64_t rows;
  int in_features, out_features;
  const uint32_t* codes;  // [out][in / 8], low nibble first
  const void* scales;     // [out][in / group]
  const void* biases;     // the same, or null: -8 * scale
  int scale_dtype;
  int group;  // 32, 64 or 128
  void* out;  // [rows][out]
  int out_dtype;
};

cudaError_t launch_affine4_linear(const Affine4Args& a, cudaStream_t s);

}  // namespace exlr8
