// Latent attention: the write into the paged cache (latent_append.cu), the
// absorbed form over it (latent_attention.cu) and the expanded form over
// per-head keys and values (latent_prompt.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace exlr8 {

constexpr int kLatentRope = 64;      // rotary channels of a key
constexpr int kLatentMaxRank = 512;  // latent channels: 128, 256, 384 or 512

struct LatentAppendArgs {
  const void* latent;  // [tokens] rows of rank, latent_stride elements apart
  int64_t latent_stride;
  const void* rope_key;  // [tokens] rows of 64
  int64_t rope_stride;
  int64_t tokens;
  int rank, dtype;
  const void* weight;  // [rank] or null: no norm
  float eps;
  const float* cos_sin;  // [cos_rows][32][2] or null: no rotation
  int64_t cos_rows;
  const int32_t* positions;
  int interleaved;
  const int64_t* slots;
  void* cache;  // [cache_rows][rank + 64]
  int64_t cache_rows;
  const void* q_rope;  // [tokens][heads] rows of 64, or null
  int64_t q_token_stride, q_head_stride;
  int heads;
  void* q_out;  // [tokens][heads][64]
};
cudaError_t launch_latent_append(const LatentAppendArgs& a, cudaStream_t s);

struct LatentAttentionArgs {
  const void *q_latent, *q_rope;  // [batch][queries][heads][rank], [...][64]
  int64_t batch;
  int queries, heads, rank, dtype;
  const void* cache;  // [pages][page_size][rank + 64]
  int64_t pages;
  int page_size;
  const int32_t* block_table;  // [batch][table_width]
  int table_width;
  const int32_t* lengths;  // [batch]
  float scale;
  void* out;   // [batch][queries][heads][rank]
  float* lse;  // [batch][queries][heads] or null
  void* workspace;
};
size_t latent_attention_workspace(int64_t batch, int queries, int heads, int rank);
cudaError_t launch_latent_attention(const LatentAttentionArgs& a, cudaStream_t s);

struct LatentPromptArgs {
  const void *q, *k, *k_rope, *v;  // element strides per token and head; channels are contiguous
  int64_t q_token, q_head, k_token, k_head, kr_token, v_token, v_head;
  int64_t total_q, total_k;
  int heads, nope, value, dtype;
  const int32_t *q_starts, *k_starts;  // [seqs + 1]
  int seqs;
  float scale;
  void* out;   // [total_q][heads][value]
  float* lse;  // [total_q][heads] or null
};
cudaError_t launch_latent_prompt(const LatentPromptArgs& a, cudaStream_t s);

}  // namespace exlr8
