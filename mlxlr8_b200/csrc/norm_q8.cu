// Residual add + RMS norm whose output is E4M3 codes with one float32 scale
// per group of channels:
//   h     = T(x + residual)
//   y     = h * (1 / sqrt(sum(h * h) / hidden + eps)) * w        (float32)
//   scale = max|y| / 448 over the group,  code = e4m3(y / scale)
// The sum of squares, the maxima and y itself stay in float32: the only
// roundings are h (an output in the activation type, as in norm.cu) and the
// code, which saturates at 448 by construction.  A group of zeros has scale 0
// and codes 0; a group with a value that is not finite has scale NaN and
// codes 0, so that every value it stands for is NaN.  A scale below the smallest
// float32 is 0, and its codes with it.
//
// Bound by memory: 8192 x 6144 bfloat16 with residual and groups of 128, 354 MB,
// 61.7 us or 5.7 TB/s; one scale a row 52.7 us; one row 2.2 us, a launch.

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

// The codes come from h w and its largest magnitude t over the group, the scale
// from t inv: 448 / t is infinite for t below 2^-119, and h w may leave float32's
// range where h inv w does not.  Where t is outside [2^-100, the largest float],
// and not 0, h is lifted by this power of two before the product with w, and
// the scale takes it back.  (|h| is below 2^64 or the sum of its squares
// infinite; then inv is 0 and the product with it is the formula's own.)
__device__ __forceinline__ bool outside(float t) {
  constexpr uint32_t kLeast = (127 - 100) << 23, kInfinity = 0x7f800000;
  // (the common answer takes one comparison; zeros and NaN are not lifted)
  return __float_as_uint(t) - kLeast >= kInfinity - kLeast && t > 0.0f;
}
__device__ __forceinline__ float lift_of(float t, float inv) {
  return inv == 0.0f ? 0.0f : t < 1.0f ? 0x1p64f : 0x1p-64f;
}
__device__ __forceinline__ float unlift_of(float t) { return t < 1.0f ? 0x1p-64f : 0x1p64f; }

// Eight channels as stored: four words of two 16-bit values, or eight floats.
template <int kAct>
struct Eight {
  uint32_t v[kAct == kF32 ? 8 : 4];
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + at * (kAct == kF32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (kAct == kF32 ? 2 : 1); ++i) {
      const uint4 u = src[i];
      v[4 * i] = u.x, v[4 * i + 1] = u.y, v[4 * i + 2] = u.z, v[4 * i + 3] = u.w;
    }
  }
  __device__ __forceinline__ void store(void* p, int64_t at) const {
    uint4* dst = reinterpret_cast<uint4*>(static_cast<char*>(p) + at * (kAct == kF32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (kAct == kF32 ? 2 : 1); ++i)
      dst[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (uint32_t& u : v) u = 0;
  }
  // The sum, rounded once to the type.
  __device__ __forceinline__ void add(const Eight& o) {
#pragma unroll
    for (int i = 0; i < (kAct == kF32 ? 8 : 4); ++i) {
      if (kAct == kF32) v[i] = __float_as_uint(__uint_as_float(v[i]) + __uint_as_float(o.v[i]));
      else if (kAct == kF16) asm("add.rn.f16x2 %0, %1, %2;" : "=r"(v[i]) : "r"(v[i]), "r"(o.v[i]));
      else asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(v[i]) : "r"(v[i]), "r"(o.v[i]));
    }
  }
  __device__ __forceinline__ float at(int i) const {
    if (kAct == kF32) return __uint_as_float(v[i]);
    const uint32_t u = v[i / 2];
    if (kAct == kBF16) return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
    return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? u >> 16 : u & 0xffffu)));
  }
};

// One row per CTA, kVecs vectors of eight channels a thread, all kept in
// registers between the sum of squares and the codes: each input is read
// once.  A group is 4, 8 or 16 lanes of one vector index, or (kWhole) the row.
// The code of y = h inv w is that of h w over its own maximum, so inv enters the
// scale alone.
template <int kAct, int kVecs, bool kWhole>
__global__ void __launch_bounds__(kVecs == 4 ? 512 : 1024)
    residual_rms_q8_kernel(const void* __restrict__ x, const void* __restrict__ residual, const void* __restrict__ w,
                           int hidden, int group, float eps, void* __restrict__ h_out, uint8_t* __restrict__ codes,
                           float* __restrict__ scales) {
  __shared__ float red[2][32];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, vecs = hidden / 8;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * hidden;
  Eight<kAct> h[kVecs], r[kVecs], f[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    if (v < vecs) {
      h[i].load(x, base + 8 * v);
      if (residual) r[i].load(residual, base + 8 * v);
      f[i].load(w, 8 * v);
    } else {
      h[i].zero();
      r[i].zero();
      f[i].zero();
    }
  }
  float acc = 0.0f;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    if (residual) h[i].add(r[i]);
    if (h_out && v < vecs) h[i].store(h_out, base + 8 * v);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = fmaf(h[i].at(e), h[i].at(e), acc);
  }
  float y[kVecs][8], top[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    top[i] = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[i][e] = h[i].at(e) * f[i].at(e);
      top[i] = max_nan(top[i], fabsf(y[i][e]));
    }
    if (!kWhole) {
#pragma unroll
      for (int off = 8; off > 0; off >>= 1)
        if (off <= group >> 4) top[i] = max_nan(top[i], __shfl_xor_sync(0xffffffffu, top[i], off));
    }
  }
  if (kWhole) {
#pragma unroll
    for (int i = 1; i < kVecs; ++i) top[0] = max_nan(top[0], top[i]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top[0] = max_nan(top[0], __shfl_xor_sync(0xffffffffu, top[0], off));
    if (lane == 0) red[1][threadIdx.x >> 5] = top[0];
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
  if (lane == 0) red[0][threadIdx.x >> 5] = acc;
  __syncthreads();
  acc = lane < warps ? red[0][lane] : 0.0f;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
  const float inv = 1.0f / sqrtf(acc / static_cast<float>(hidden) + eps);
  if (kWhole) {
    top[0] = lane < warps ? red[1][lane] : 0.0f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top[0] = max_nan(top[0], __shfl_xor_sync(0xffffffffu, top[0], off));
  }
  // The products of vector i again, h lifted, from the inputs; their largest.
  auto lifted = [&](int i, float lift) {
    const int v = i * blockDim.x + threadIdx.x;
    float most = 0.0f;
    if (v < vecs) {
      Eight<kAct> sum, other;
      sum.load(x, base + 8 * v);
      if (residual) {
        other.load(residual, base + 8 * v);
        sum.add(other);
      }
      other.load(w, 8 * v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[i][e] = sum.at(e) * lift * other.at(e);
        most = max_nan(most, fabsf(y[i][e]));
      }
    }
    return most;
  };
  float unlift[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) unlift[i] = 1.0f;
  if (kWhole && outside(top[0])) {  // the same for all threads
    const float lift = lift_of(top[0], inv);
    unlift[0] = unlift_of(top[0]);
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) most = max_nan(most, lifted(i, lift));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, off));
    __syncthreads();  // the maxima of the products are read
    if (lane == 0) red[1][threadIdx.x >> 5] = most;
    __syncthreads();
    top[0] = lane < warps ? red[1][lane] : 0.0f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top[0] = max_nan(top[0], __shfl_xor_sync(0xffffffffu, top[0], off));
  }
  const int lanes = group >> 3;  // threads of a group
  bool some = false;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) some = some || outside(top[i]);
  if (!kWhole && some) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      if (!outside(top[i])) continue;  // the same for the group's threads
      const uint32_t mask = ((1u << lanes) - 1) << (lane & ~(lanes - 1));
      unlift[i] = unlift_of(top[i]);
      top[i] = lifted(i, lift_of(top[i], inv));
      for (int off = lanes / 2; off > 0; off >>= 1) top[i] = max_nan(top[i], __shfl_xor_sync(mask, top[i], off));
    }
  }
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    if (v >= vecs) continue;
    const float t = kWhole ? top[0] : top[i];
    // inv is 0 in a row with an infinity, NaN in one with a NaN.
    const float scale = t * inv / 448.0f * unlift[kWhole ? 0 : i];
    const bool finite = t < __int_as_float(0x7f800000) && scale < __int_as_float(0x7f800000);
    const float mul = scale > 0.0f && finite ? 448.0f / t : 0.0f;
    uint32_t two[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint16_t c;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(y[i][2 * e + 1] * mul), "f"(y[i][2 * e] * mul));
      two[e] = c;
    }
    const uint2 out = finite ? make_uint2(two[0] | two[1] << 16, two[2] | two[3] << 16) : make_uint2(0, 0);
    *reinterpret_cast<uint2*>(codes + base + 8 * v) = out;
    if (kWhole ? v == 0 : threadIdx.x % lanes == 0)
      scales[kWhole ? blockIdx.x : base / group + v / lanes] = finite ? scale : __int_as_float(0x7fc00000);
  }
}

// One CTA per row, any hidden size and alignment.  kCached keeps h w of the row
// in shared memory, so that the inputs are read once; rows beyond kCachedMax
// channels read them again.  Single loads: 5000 x 7999 bfloat16 85 us, 3.3 TB/s
// (106 us with the inputs read three times).
constexpr int kCachedMax = 24 * 1024;  // two CTAs of 96 KB per SM

template <int kAct, bool kCached>
__global__ void __launch_bounds__(kThreads) residual_rms_q8_any_kernel(const void* __restrict__ x,
                                                                       const void* __restrict__ residual,
                                                                       const void* __restrict__ w, int hidden,
                                                                       int group, float eps, void* __restrict__ h_out,
                                                                       uint8_t* __restrict__ codes,
                                                                       float* __restrict__ scales) {
  extern __shared__ float cache[];
  __shared__ float red[2][kThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * hidden;
  auto sum_at = [&](int i) {
    const float h = load_act(x, kAct, base + i);
    return residual ? round_to(kAct, h + load_act(residual, kAct, base + i)) : h;
  };
  float lift = 1.0f;
  auto weighted = [&](int i) { return kCached ? cache[i] : sum_at(i) * lift * load_act(w, kAct, i); };
  float acc = 0.0f, row_top = 0.0f;
#pragma unroll 4
  for (int i = threadIdx.x; i < hidden; i += kThreads) {
    const float h = sum_at(i), y = h * load_act(w, kAct, i);
    if (kCached) cache[i] = y;
    if (h_out) store_act(h_out, kAct, base + i, h);
    acc = fmaf(h, h, acc);
    row_top = max_nan(row_top, fabsf(y));
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    acc += __shfl_xor_sync(0xffffffffu, acc, off);
    row_top = max_nan(row_top, __shfl_xor_sync(0xffffffffu, row_top, off));
  }
  if (lane == 0) {
    red[0][warp] = acc;
    red[1][warp] = row_top;
  }
  __syncthreads();
  acc = row_top = 0.0f;
  for (int i = 0; i < kThreads / 32; ++i) {
    acc += red[0][i];
    row_top = max_nan(row_top, red[1][i]);
  }
  const float inv = 1.0f / sqrtf(acc / static_cast<float>(hidden) + eps);
  const int groups = hidden / group;
  // A warp takes whole groups; all threads share the one group of a row.
  for (int gi = groups == 1 ? 0 : warp; gi < groups; gi += kThreads / 32) {
    float top = row_top;
    if (groups > 1) {
      top = 0.0f;
      for (int i = lane; i < group; i += 32) top = max_nan(top, fabsf(weighted(gi * group + i)));
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
    }
    const int first = groups == 1 ? threadIdx.x : lane, step = groups == 1 ? kThreads : 32;
    float unlift = 1.0f;
    if (outside(top)) {  // the same for the threads of a group
      lift = lift_of(top, inv);
      unlift = unlift_of(top);
      top = 0.0f;
      for (int i = gi * group + first; i < (gi + 1) * group; i += step) {
        const float y = sum_at(i) * lift * load_act(w, kAct, i);
        if (kCached) cache[i] = y;
        top = max_nan(top, fabsf(y));
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
      if (groups == 1) {
        __syncthreads();  // the maxima of the products are read
        if (lane == 0) red[1][warp] = top;
        __syncthreads();
        for (int i = 0; i < kThreads / 32; ++i) top = max_nan(top, red[1][i]);
      }
    }
    const float scale = top * inv / 448.0f * unlift;
    const bool finite = top < __int_as_float(0x7f800000) && scale < __int_as_float(0x7f800000);
    const float mul = scale > 0.0f && finite ? 448.0f / top : 0.0f;
#pragma unroll 4
    for (int i = gi * group + first; i < (gi + 1) * group; i += step)
      codes[base + i] = finite ? to_e4m3(weighted(i) * mul) : 0;
    if (groups == 1 ? threadIdx.x == 0 : lane == 0)
      scales[static_cast<int64_t>(blockIdx.x) * groups + gi] = finite ? scale : __int_as_float(0x7fc00000);
    lift = 1.0f;
  }
}

template <int kAct, int kVecs>
cudaError_t launch_vectors(const void* x, const void* residual, const void* w, int64_t rows, int hidden, int group,
                           float eps, void* h_out, uint8_t* codes, float* scales, cudaStream_t s) {
  const int vecs = hidden / 8, threads = ((vecs + kVecs - 1) / kVecs + 31) / 32 * 32;
  const dim3 grid(static_cast<unsigned>(rows)), block(threads);
  if (group == hidden)
    return launch_pdl(residual_rms_q8_kernel<kAct, kVecs, true>, grid, block, 0, s, x, residual, w, hidden, group, eps,
                      h_out, codes, scales);
  return launch_pdl(residual_rms_q8_kernel<kAct, kVecs, false>, grid, block, 0, s, x, residual, w, hidden, group, eps,
                    h_out, codes, scales);
}

template <int kAct>
cudaError_t launch(const void* x, const void* residual, const void* w, int64_t rows, int hidden, int group, float eps,
                   void* h_out, uint8_t* codes, float* scales, cudaStream_t s) {
  auto aligned = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  const bool vectors = hidden % 8 == 0 && aligned(x, 16) && aligned(residual, 16) && aligned(w, 16) &&
                       aligned(h_out, 16) && aligned(codes, 8);
  // A few rows spread over as many threads as a row has vectors; many rows
  // leave more loads to a thread and more rows to an SM.  296: two CTAs an SM.
  const int vecs = hidden / 8;
  const bool few = rows <= 296;
  if (vectors && vecs <= (few ? 1024 : 256))
    return launch_vectors<kAct, 1>(x, residual, w, rows, hidden, group, eps, h_out, codes, scales, s);
  if (vectors && vecs <= (few ? 2048 : 512))
    return launch_vectors<kAct, 2>(x, residual, w, rows, hidden, group, eps, h_out, codes, scales, s);
  if (vectors && !few && vecs <= 2048)
    return launch_vectors<kAct, 4>(x, residual, w, rows, hidden, group, eps, h_out, codes, scales, s);
  const dim3 grid(static_cast<unsigned>(rows));
  if (hidden > kCachedMax)
    return launch_pdl(residual_rms_q8_any_kernel<kAct, false>, grid, dim3(kThreads), 0, s, x, residual, w, hidden,
                      group, eps, h_out, codes, scales);
  static std::atomic<uint64_t> ready{0};
  const cudaError_t err = allow_shared_memory(residual_rms_q8_any_kernel<kAct, true>, kCachedMax * 4, ready);
  if (err != cudaSuccess) return err;
  return launch_pdl(residual_rms_q8_any_kernel<kAct, true>, grid, dim3(kThreads), static_cast<size_t>(hidden) * 4, s, x,
                    residual, w, hidden, group, eps, h_out, codes, scales);
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
