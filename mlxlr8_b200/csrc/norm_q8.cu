// Residual add + RMS norm whose output is E4M3 codes with one float32 scale
// per group of channels:
//   h     = T(x + residual)
//   y     = h * (1 / sqrt(sum(h * h) / hidden + eps)) * w        (float32)
//   scale = max|y| / 448 over the group,  code = e4m3(y / scale)
// The sum of squares, the maxima and y itself stay in float32: the only
// roundings are h (an output in the activation type, as in norm.cu) and the
// code, which saturates at 448 by construction.  A group of zeros has scale 0
// and codes 0; a group with a value that is not finite has scale NaN and
// codes 0, so that every value it stands for is NaN.

#include "common.cuh"
#include "launch.cuh"
#include "norm_q8.cuh"

namespace exlr8 {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint8_t to_e4m3(float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
  return static_cast<uint8_t>(r);
}

// max(|a|) that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// One CTA per row, any hidden size and alignment.
template <int kAct>
__global__ void __launch_bounds__(kThreads) residual_rms_q8_any_kernel(const void* __restrict__ x,
                                                                       const void* __restrict__ residual,
                                                                       const void* __restrict__ w, int hidden,
                                                                       int group, float eps, void* __restrict__ h_out,
                                                                       uint8_t* __restrict__ codes,
                                                                       float* __restrict__ scales) {
  __shared__ float red[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * hidden;
  auto value = [&](int i) {
    const float h = load_act(x, kAct, base + i);
    return residual ? round_to(kAct, h + load_act(residual, kAct, base + i)) : h;
  };
  float acc = 0.0f;
  for (int i = threadIdx.x; i < hidden; i += kThreads) {
    const float h = value(i);
    if (h_out) store_act(h_out, kAct, base + i, h);
    acc = fmaf(h, h, acc);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
  if (lane == 0) red[warp] = acc;
  __syncthreads();
  acc = 0.0f;
  for (int i = 0; i < kThreads / 32; ++i) acc += red[i];
  const float inv = 1.0f / sqrtf(acc / static_cast<float>(hidden) + eps);
  const int groups = hidden / group;
  // A warp takes whole groups; with one group a row every warp finds its
  // maximum again.
  for (int gi = groups == 1 ? 0 : warp; gi < groups; gi += kThreads / 32) {
    float top = 0.0f;
    for (int i = lane; i < group; i += 32)
      top = max_nan(top, fabsf(value(gi * group + i) * inv * load_act(w, kAct, gi * group + i)));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
    const bool finite = top < __int_as_float(0x7f800000);
    const float mul = finite && top > 0.0f ? 448.0f / top : 0.0f;
    const int first = groups == 1 ? threadIdx.x : lane, step = groups == 1 ? kThreads : 32;
    for (int i = first; i < group; i += step) {
      const float y = value(gi * group + i) * inv * load_act(w, kAct, gi * group + i);
      codes[base + gi * group + i] = finite ? to_e4m3(y * mul) : 0;
    }
    if (groups == 1 ? threadIdx.x == 0 : lane == 0)
      scales[static_cast<int64_t>(blockIdx.x) * groups + gi] = finite ? top / 448.0f : __int_as_float(0x7fc00000);
  }
}

template <int kAct>
cudaError_t launch(const void* x, const void* residual, const void* w, int64_t rows, int hidden, int group, float eps,
                   void* h_out, uint8_t* codes, float* scales, cudaStream_t s) {
  residual_rms_q8_any_kernel<kAct><<<static_cast<unsigned>(rows), kThreads, 0, s>>>(x, residual, w, hidden, group, eps,
                                                                                   h_out, codes, scales);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_residual_rms_q8(const void* x, const void* residual, const void* w, int act_dtype, int64_t rows,
                                   int hidden, int group, float eps, void* h_out, uint8_t* codes, float* scales,
                                   cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  if (act_dtype == kF32) return launch<kF32>(x, residual, w, rows, hidden, group, eps, h_out, codes, scales, s);
  if (act_dtype == kF16) return launch<kF16>(x, residual, w, rows, hidden, group, eps, h_out, codes, scales, s);
  return launch<kBF16>(x, residual, w, rows, hidden, group, eps, h_out, codes, scales, s);
}

}  // namespace exlr8
