// y[t][o] = sum_g s[o][g] * sum_{k in g} q[o][k] x[t][k] + b[o][g] * sum_{k in g} x[t][k]
// over 4-bit codes q (eight per uint32, low nibble first), group scales s and
// biases b (b = -8 s without them).  The sums run over q - 8, which halves
// what cancels, with b + 8 s in place of b; all sums are float32.

#include "affine4.cuh"
#include "common.cuh"

namespace exlr8 {

namespace {

__device__ __forceinline__ float load_x(const void* x, int dtype, int64_t i) {
  if (dtype != EXLR8_DTYPE_E4M3) return load_act(x, dtype, i);
  uint32_t h2;
  const uint16_t code = static_cast<const uint8_t*>(x)[i];
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(code));
  return __half2float(__ushort_as_half(static_cast<unsigned short>(h2 & 0xffffu)));
}

// One warp per output and row.
__global__ void __launch_bounds__(256) affine4_rows_kernel(const Affine4Args a) {
  const int lane = threadIdx.x & 31;
  const int o = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (o >= a.out_features) return;
  const int words = a.in_features / 8, groups = a.in_features / a.group;
  for (int64_t t = blockIdx.y; t < a.rows; t += gridDim.y) {
    float acc = 0.0f;
    for (int i = lane; i < words; i += 32) {
      const uint32_t w = a.codes[static_cast<int64_t>(o) * words + i];
      const int64_t at = t * a.in_features + 8 * i;
      float dot = 0.0f, sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = load_x(a.x, a.x_dtype, at + j);
        dot = fmaf(static_cast<float>(static_cast<int>((w >> (4 * j)) & 15u) - 8), v, dot);
        sum += v;
      }
      const int64_t g = static_cast<int64_t>(o) * groups + 8 * i / a.group;
      const float s = load_act(a.scales, a.scale_dtype, g);
      float part = s * dot;
      if (a.biases) part = fmaf(fmaf(8.0f, s, load_act(a.biases, a.scale_dtype, g)), sum, part);
      if (a.x_scales) part *= a.x_scales[t * (a.in_features / a.x_group) + 8 * i / a.x_group];
      acc += part;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    if (lane == 0) store_act(a.out, a.out_dtype, t * a.out_features + o, acc);
  }
}

}  // namespace

cudaError_t launch_affine4_linear(const Affine4Args& a, cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  const dim3 grid((a.out_features + 7) / 8, static_cast<unsigned>(a.rows < 1024 ? a.rows : 1024));
  affine4_rows_kernel<<<grid, 256, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace exlr8
