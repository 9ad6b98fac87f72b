// One token's entry into the paged latent cache and the rotation of its
// queries:
//   cache[slot] = [T(c * (1 / sqrt(sum(c * c) / rank + eps)) * w), T(rot(k))]
//   q_out[h]    = T(rot(q[h]))
//   rot(a, b)   = (a cos - b sin, a sin + b cos)
// for the pairs (2i, 2i + 1), or (i, i + 32) when not interleaved, with the
// table's cosine and sine of the token's position; float32 throughout, one
// rounding at the store.  A token whose slot is outside the cache (a padding
// row carries -1) writes no entry; a position outside the table writes no
// entry and NaN queries.
//
// Bound by memory: 8192 tokens of rank 512 with the queries of 64 heads, 155 MB,
// 31 us or 5.0 TB/s; 32 tokens 2.2 us, a launch.  (Queries fetched ahead of the
// position: 30.3 and 2.4 us.)

#include "common.cuh"
#include "latent.cuh"
#include "launch.cuh"

namespace exlr8 {

namespace {

constexpr int kThreads = 256;

// Eight channels as float32 and back.
template <int kAct>
__device__ __forceinline__ void load8(const void* p, int64_t at, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
  const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (kAct == kBF16) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

template <int kAct>
__device__ __forceinline__ void store8(void* p, int64_t at, const float (&v)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = pack<kAct>(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at) = make_uint4(u[0], u[1], u[2], u[3]);
}

constexpr int kVecThreads = 128;

// One CTA per token, 16-byte accesses: warp 0 takes the latent (eight or
// sixteen channels a lane, so its sum needs no barrier) and the key, the other
// warps the queries.  A rotation item is eight pairs: two vectors of one row,
// adjacent when interleaved, 32 channels apart when not; an item's pairs
// depend on the thread alone, so their cosines are read once for all heads.
template <int kAct>
__global__ void __launch_bounds__(kVecThreads) latent_append_vec_kernel(const LatentAppendArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t slot = a.slots[t];
  const int position = a.cos_sin ? a.positions[t] : 0;
  const bool known = !a.cos_sin || (position >= 0 && position < a.cos_rows);
  const bool store = known && slot >= 0 && slot < a.cache_rows;
  const int64_t row = slot * (a.rank + kLatentRope);
  const int v = threadIdx.x & 3;
  float c[8], n[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = known ? 1.0f : __int_as_float(0x7fc00000);
    n[i] = 0.0f;
  }
  if (a.cos_sin && known) {
    const float4* table = reinterpret_cast<const float4*>(a.cos_sin + (static_cast<int64_t>(position) * 32 + 8 * v) * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 f = table[i];
      c[2 * i] = f.x, n[2 * i] = f.y, c[2 * i + 1] = f.z, n[2 * i + 1] = f.w;
    }
  }
  const int first = a.interleaved ? 16 * v : 8 * v, second = a.interleaved ? 16 * v + 8 : 32 + 8 * v;
  auto rotate = [&](const void* src, int64_t from, void* dst, int64_t to) {
    if (!a.cos_sin) {  // (0 times an infinity would reach the pair's other channel)
      auto* const at = static_cast<uint16_t*>(dst) + to;
      auto* const of = static_cast<const uint16_t*>(src) + from;
      *reinterpret_cast<uint4*>(at + first) = *reinterpret_cast<const uint4*>(of + first);
      *reinterpret_cast<uint4*>(at + second) = *reinterpret_cast<const uint4*>(of + second);
      return;
    }
    float x[8], y[8];
    load8<kAct>(src, from + first, x);
    load8<kAct>(src, from + second, y);
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float p = x[i], q = x[i + 1], r = y[i], s = y[i + 1];
        x[i] = p * c[i / 2] - q * n[i / 2];
        x[i + 1] = p * n[i / 2] + q * c[i / 2];
        y[i] = r * c[4 + i / 2] - s * n[4 + i / 2];
        y[i + 1] = r * n[4 + i / 2] + s * c[4 + i / 2];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = x[i], q = y[i];
        x[i] = p * c[i] - q * n[i];
        y[i] = p * n[i] + q * c[i];
      }
    }
    store8<kAct>(dst, to + first, x);
    store8<kAct>(dst, to + second, y);
  };
  if (warp == 0) {
    if (!store) return;
    float x[2][8];
    float acc = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = 8 * (lane + 32 * i);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = 0.0f;
      if (at < a.rank) load8<kAct>(a.latent, t * a.latent_stride + at, x[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc = fmaf(x[i][e], x[i][e], acc);
    }
    if (lane < 4) rotate(a.rope_key, t * a.rope_stride, a.cache, row + a.rank);
    if (a.weight) {
      __syncwarp();
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
      const float inv = 1.0f / sqrtf(acc / static_cast<float>(a.rank) + a.eps);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = 8 * (lane + 32 * i);
        if (at >= a.rank) continue;
        float f[8];
        load8<kAct>(a.weight, at, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = x[i][e] * inv * f[e];
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = 8 * (lane + 32 * i);
      if (at < a.rank) store8<kAct>(a.cache, row + at, x[i]);
    }
  } else if (a.q_rope) {
#pragma unroll 2
    for (int h = (threadIdx.x - 32) >> 2; h < a.heads; h += (kVecThreads - 32) / 4)
      rotate(a.q_rope, t * a.q_token_stride + h * a.q_head_stride, a.q_out, (t * a.heads + h) * kLatentRope);
  }
}

// One CTA per token, any strides and alignment.
template <int kAct>
__global__ void __launch_bounds__(kThreads) latent_append_kernel(const LatentAppendArgs a) {
  __shared__ float red[kThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = blockIdx.x;
  const int64_t slot = a.slots[t];
  const int position = a.cos_sin ? a.positions[t] : 0;
  const bool known = !a.cos_sin || (position >= 0 && position < a.cos_rows);
  const bool store = known && slot >= 0 && slot < a.cache_rows;
  float inv = 1.0f;
  if (a.weight) {
    float acc = 0.0f;
    for (int i = threadIdx.x; i < a.rank; i += kThreads) {
      const float v = load_act(a.latent, kAct, t * a.latent_stride + i);
      acc = fmaf(v, v, acc);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = acc;
    __syncthreads();
    acc = 0.0f;
    for (int i = 0; i < kThreads / 32; ++i) acc += red[i];
    inv = 1.0f / sqrtf(acc / static_cast<float>(a.rank) + a.eps);
  }
  const int64_t row = slot * (a.rank + kLatentRope);
  if (store) {
    for (int i = threadIdx.x; i < a.rank; i += kThreads) {
      float v = load_act(a.latent, kAct, t * a.latent_stride + i);
      if (a.weight) v = v * inv * load_act(a.weight, kAct, i);
      store_act(a.cache, kAct, row + i, v);
    }
  }
  // Pair p of head h: item h * 32 + p; the key is head -1.
  const int items = 32 * ((a.q_rope ? a.heads : 0) + 1);
  for (int i = threadIdx.x; i < items; i += kThreads) {
    const int h = i / 32 - 1, p = i % 32;
    const int first = a.interleaved ? 2 * p : p, second = a.interleaved ? 2 * p + 1 : p + 32;
    const void* src = h < 0 ? a.rope_key : a.q_rope;
    const int64_t at = h < 0 ? t * a.rope_stride : t * a.q_token_stride + h * a.q_head_stride;
    const float u = load_act(src, kAct, at + first), v = load_act(src, kAct, at + second);
    float c = 1.0f, n = 0.0f;
    if (a.cos_sin) {
      c = known ? a.cos_sin[(static_cast<int64_t>(position) * 32 + p) * 2] : __int_as_float(0x7fc00000);
      n = known ? a.cos_sin[(static_cast<int64_t>(position) * 32 + p) * 2 + 1] : 0.0f;
    }
    // (without a table 0 times an infinity would reach the pair's other channel)
    const float x = a.cos_sin ? u * c - v * n : u, y = a.cos_sin ? u * n + v * c : v;
    if (h < 0) {
      if (store) {
        store_act(a.cache, kAct, row + a.rank + first, x);
        store_act(a.cache, kAct, row + a.rank + second, y);
      }
    } else {
      const int64_t to = (t * a.heads + h) * kLatentRope;
      store_act(a.q_out, kAct, to + first, x);
      store_act(a.q_out, kAct, to + second, known ? y : c);
    }
  }
}

}  // namespace

cudaError_t launch_latent_append(const LatentAppendArgs& a, cudaStream_t s) {
  if (a.tokens == 0) return cudaSuccess;
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vectors = aligned(a.latent) && aligned(a.rope_key) && aligned(a.weight) && aligned(a.cos_sin) &&
                       aligned(a.cache) && aligned(a.q_rope) && aligned(a.q_out) && a.latent_stride % 8 == 0 &&
                       a.rope_stride % 8 == 0 && a.q_token_stride % 8 == 0 && a.q_head_stride % 8 == 0;
  const dim3 grid(static_cast<unsigned>(a.tokens));
  if (vectors)
    return launch_pdl(a.dtype == kF16 ? latent_append_vec_kernel<kF16> : latent_append_vec_kernel<kBF16>, grid,
                      dim3(kVecThreads), 0, s, a);
  return launch_pdl(a.dtype == kF16 ? latent_append_kernel<kF16> : latent_append_kernel<kBF16>, grid, dim3(kThreads), 0,
                    s, a);
}

}  // namespace exlr8
