// Causal attention of ragged prompts over expanded keys and values: head h of
// key j is [k_j,h, k_rope_j] (the rotary part is shared by all heads) and its
// value v_j,h.  Query i of a sequence with n queries and m keys sees its
// first m - n + 1 + i keys, so a chunk with a history ends with its keys.  A
// query that sees none gives zeros (and lse -inf).  Statistics in float32.

#include "common.cuh"
#include "latent.cuh"

namespace exlr8 {

namespace {

constexpr int kWarps = 4;

// The sequence of query `row`, or -1 (a row behind the last sequence).
__device__ __forceinline__ int sequence_of(const int32_t* starts, int seqs, int64_t row) {
  for (int s = 0; s < seqs; ++s)
    if (row >= starts[s] && row < starts[s + 1]) return s;
  return -1;
}

// One CTA per query and head; a warp takes every fourth key.
template <int kAct>
__global__ void __launch_bounds__(32 * kWarps) latent_prompt_kernel(const LatentPromptArgs a) {
  __shared__ float s_m[kWarps], s_l[kWarps], s_o[kWarps][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const int h = blockIdx.y;
  const int seq = sequence_of(a.q_starts, a.seqs, row);
  if (seq < 0) return;
  const int64_t k0 = min(static_cast<int64_t>(max(a.k_starts[seq], 0)), a.total_k);
  const int64_t k1 = min(static_cast<int64_t>(a.k_starts[seq + 1]), a.total_k);
  const int64_t queries = a.q_starts[seq + 1] - a.q_starts[seq];
  const int64_t seen = k1 - k0 - queries + 1 + (row - a.q_starts[seq]);
  const int nb = a.nope / 64, vb = a.value / 64;
  float q[8], o[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    for (int e = 0; e < 2; ++e) {
      q[2 * i + e] =
          i <= nb ? load_act(a.q, kAct, row * a.q_token + h * a.q_head + 64 * i + 2 * lane + e) : 0.0f;
      o[2 * i + e] = 0.0f;
    }
  }
  float m = -INFINITY, l = 0.0f;
  for (int64_t j = warp; j < seen; j += kWarps) {
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      for (int e = 0; e < 2; ++e) {
        float k = 0.0f;
        if (i < nb) k = load_act(a.k, kAct, (k0 + j) * a.k_token + h * a.k_head + 64 * i + 2 * lane + e);
        else if (i == nb) k = load_act(a.k_rope, kAct, (k0 + j) * a.kr_token + 2 * lane + e);
        dot = fmaf(q[2 * i + e], k, dot);
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    const float s = dot * a.scale;
    const float top = fmaxf(m, s);
    if (top == -INFINITY) continue;
    const float keep = expf(m - top), p = expf(s - top);
    m = top;
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      for (int e = 0; e < 2; ++e) {
        if (i >= vb) continue;
        const float v = load_act(a.v, kAct, (k0 + j) * a.v_token + h * a.v_head + 64 * i + 2 * lane + e);
        o[2 * i + e] = fmaf(p, v, o[2 * i + e] * keep);
      }
    }
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s_o[warp][64 * i + 2 * lane] = o[2 * i];
    s_o[warp][64 * i + 2 * lane + 1] = o[2 * i + 1];
  }
  __syncthreads();
  float top = -INFINITY, sum = 0.0f;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w]);
  for (int w = 0; w < kWarps; ++w) sum += s_l[w] > 0.0f ? s_l[w] * expf(s_m[w] - top) : 0.0f;
  for (int i = threadIdx.x; i < a.value; i += 32 * kWarps) {
    float v = 0.0f;
    for (int w = 0; w < kWarps; ++w) v += s_l[w] > 0.0f ? s_o[w][i] * expf(s_m[w] - top) : 0.0f;
    store_act(a.out, kAct, (row * a.heads + h) * a.value + i, sum > 0.0f ? v / sum : 0.0f);
  }
  if (a.lse && threadIdx.x == 0) a.lse[row * a.heads + h] = sum > 0.0f ? top + logf(sum) : -INFINITY;
}

}  // namespace

cudaError_t launch_latent_prompt(const LatentPromptArgs& a, cudaStream_t s) {
  if (a.total_q == 0 || a.seqs == 0) return cudaSuccess;
  const dim3 grid(static_cast<unsigned>(a.total_q), a.heads);
  if (a.dtype == kF16) latent_prompt_kernel<kF16><<<grid, 32 * kWarps, 0, s>>>(a);
  else latent_prompt_kernel<kBF16><<<grid, 32 * kWarps, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace exlr8
