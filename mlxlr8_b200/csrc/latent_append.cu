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

#include "common.cuh"
#include "latent.cuh"

namespace exlr8 {

namespace {

constexpr int kThreads = 256;

// One CTA per token.
template <int kAct>
__global__ void __launch_bounds__(kThreads) latent_append_kernel(const LatentAppendArgs a) {
  __shared__ float red[kThreads / 32];
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
    const float x = u * c - v * n, y = u * n + v * c;
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
  const unsigned grid = static_cast<unsigned>(a.tokens);
  if (a.dtype == kF16) latent_append_kernel<kF16><<<grid, kThreads, 0, s>>>(a);
  else latent_append_kernel<kBF16><<<grid, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace exlr8
