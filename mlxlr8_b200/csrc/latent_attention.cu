// Attention over the paged latent cache (absorbed form): every head of a
// query attends the same row [c_j, k_j] of a token,
//   s_j = scale * (ql . c_j + qr . k_j),  out = sum_j softmax(s)_j c_j,
// in one pass with the running maximum and sum of the softmax in float32.
// Query t of T sees the first length - T + 1 + t tokens; a query that sees
// none gives zeros (and lse -inf).  Table entries outside the cache hold no
// tokens.

#include "common.cuh"
#include "latent.cuh"

namespace exlr8 {

namespace {

constexpr int kWarps = 8;

// One CTA per query and head; a warp takes every eighth token, a lane two
// channels of each 64, and the warps' states join in shared memory.
template <int kAct>
__global__ void __launch_bounds__(32 * kWarps) latent_attention_kernel(const LatentAttentionArgs a) {
  __shared__ float s_m[kWarps], s_l[kWarps], s_o[kWarps][kLatentMaxRank];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const int64_t b = row / (static_cast<int64_t>(a.queries) * a.heads);
  const int t = static_cast<int>(row / a.heads % a.queries);
  const int nb = a.rank / 64;
  float q[2 * (kLatentMaxRank / 64 + 1)], o[2 * (kLatentMaxRank / 64)];
#pragma unroll
  for (int i = 0; i < kLatentMaxRank / 64 + 1; ++i) {
    for (int e = 0; e < 2; ++e)
      q[2 * i + e] = i < nb ? load_act(a.q_latent, kAct, row * a.rank + 64 * i + 2 * lane + e) : 0.0f;
  }
  const float r0 = load_act(a.q_rope, kAct, row * 64 + 2 * lane), r1 = load_act(a.q_rope, kAct, row * 64 + 2 * lane + 1);
#pragma unroll
  for (int i = 0; i < 2 * (kLatentMaxRank / 64); ++i) o[i] = 0.0f;
  const int64_t room = static_cast<int64_t>(a.table_width) * a.page_size;
  const int64_t length = min(static_cast<int64_t>(a.lengths[b]), room);
  const int64_t seen = length - a.queries + 1 + t;
  float m = -INFINITY, l = 0.0f;
  for (int64_t j = warp; j < seen; j += kWarps) {
    const int page = a.block_table[b * a.table_width + j / a.page_size];
    if (page < 0 || page >= a.pages) continue;
    const int64_t at = (static_cast<int64_t>(page) * a.page_size + j % a.page_size) * (a.rank + kLatentRope);
    float c[2 * (kLatentMaxRank / 64)];
    float dot = r0 * load_act(a.cache, kAct, at + a.rank + 2 * lane) +
                r1 * load_act(a.cache, kAct, at + a.rank + 2 * lane + 1);
#pragma unroll
    for (int i = 0; i < kLatentMaxRank / 64; ++i) {
      for (int e = 0; e < 2; ++e) {
        c[2 * i + e] = i < nb ? load_act(a.cache, kAct, at + 64 * i + 2 * lane + e) : 0.0f;
        dot = fmaf(q[2 * i + e], c[2 * i + e], dot);
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
    for (int i = 0; i < 2 * (kLatentMaxRank / 64); ++i) o[i] = fmaf(p, c[i], o[i] * keep);
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < kLatentMaxRank / 64; ++i) {
    s_o[warp][64 * i + 2 * lane] = o[2 * i];
    s_o[warp][64 * i + 2 * lane + 1] = o[2 * i + 1];
  }
  __syncthreads();
  float top = -INFINITY, sum = 0.0f;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w]);
  for (int w = 0; w < kWarps; ++w) sum += s_l[w] > 0.0f ? s_l[w] * expf(s_m[w] - top) : 0.0f;
  for (int i = threadIdx.x; i < a.rank; i += 32 * kWarps) {
    float v = 0.0f;
    for (int w = 0; w < kWarps; ++w) v += s_l[w] > 0.0f ? s_o[w][i] * expf(s_m[w] - top) : 0.0f;
    store_act(a.out, kAct, row * a.rank + i, sum > 0.0f ? v / sum : 0.0f);
  }
  if (a.lse && threadIdx.x == 0) a.lse[row] = sum > 0.0f ? top + logf(sum) : -INFINITY;
}

}  // namespace

size_t latent_attention_workspace(int64_t, int, int, int) { return 0; }

cudaError_t launch_latent_attention(const LatentAttentionArgs& a, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(a.batch * a.queries * a.heads);
  if (grid == 0) return cudaSuccess;
  if (a.dtype == kF16) latent_attention_kernel<kF16><<<grid, 32 * kWarps, 0, s>>>(a);
  else latent_attention_kernel<kBF16><<<grid, 32 * kWarps, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace exlr8
