// extern "C" entry points of the attention half of a decoder block: the 8-bit
// residual norm, the 4-bit affine linear layer, and latent attention (cache
// append, absorbed form, expanded form).  Sizes, types, strides and alignment
// are checked here on the host; what only the device knows (slots, positions,
// pages, lengths) is bounded by the kernels.

#include <cmath>
#include <initializer_list>

#include "affine4.cuh"
#include "capi_util.cuh"
#include "latent.cuh"
#include "norm_q8.cuh"

using namespace exlr8;

namespace {

bool half_type(int d) { return d == EXLR8_DTYPE_F16 || d == EXLR8_DTYPE_BF16; }
bool rank_ok(int rank) { return rank >= 128 && rank <= kLatentMaxRank && rank % 128 == 0; }
constexpr int64_t kMaxGrid = 0x7fffffff;
bool pages_ok(int64_t pages, int page_size) {
  return pages >= 0 && page_size > 0 && page_size % 16 == 0 && page_size <= (1 << 20) && pages <= kMaxGrid &&
         pages * page_size <= kMaxGrid;
}

// The bytes from an operand's first element to its last, gaps between rows
// among them; empty without a pointer.
struct Span {
  __int128 begin = 0, end = 0;
  Span(const void* p, __int128 bytes) {
    if (p == nullptr || bytes <= 0) return;
    begin = reinterpret_cast<uintptr_t>(p);
    end = begin + bytes;
  }
  // Rows of `width` 16-bit channels, [n][m] of them with element strides of
  // either sign.
  Span(const void* p, int64_t n, int64_t n_stride, int64_t m, int64_t m_stride, int width) {
    if (p == nullptr || n <= 0 || m <= 0) return;
    const __int128 a = static_cast<__int128>(n - 1) * n_stride, b = static_cast<__int128>(m - 1) * m_stride;
    begin = reinterpret_cast<uintptr_t>(p) + 2 * ((a < 0 ? a : 0) + (b < 0 ? b : 0));
    end = reinterpret_cast<uintptr_t>(p) + 2 * ((a > 0 ? a : 0) + (b > 0 ? b : 0) + width);
  }
  bool meets(const Span& o) const { return begin < o.end && o.begin < end && begin < end && o.begin < o.end; }
};
// Whether a written span meets one that is read, or another written one.
bool overlap(std::initializer_list<Span> written, std::initializer_list<Span> read) {
  for (const Span* w = written.begin(); w != written.end(); ++w) {
    for (const Span& r : read)
      if (w->meets(r)) return true;
    for (const Span* v = w + 1; v != written.end(); ++v)
      if (w->meets(*v)) return true;
  }
  return false;
}
int size_of(int dtype) { return dtype == EXLR8_DTYPE_F32 ? 4 : dtype == EXLR8_DTYPE_E4M3 ? 1 : 2; }

}  // namespace

extern "C" {

int exlr8_residual_rms_norm_q8(const void* x, const void* residual, const void* weight, int x_dtype, int64_t rows,
                               int hidden, int group, float eps, void* h_out, uint8_t* codes, float* scales,
                               void* stream) {
  if (!valid_act(x_dtype)) return EXLR8_ERR_DTYPE;
  if (rows < 0 || rows > kMaxGrid || hidden <= 0) return EXLR8_ERR_SHAPE;
  if (group != hidden && ((group != 32 && group != 64 && group != 128) || hidden % group)) return EXLR8_ERR_SHAPE;
  if (rows == 0) return EXLR8_OK;
  if (!x || !weight || !codes || !scales || !(eps >= 0.0f)) return EXLR8_ERR_ARG;
  const __int128 n = static_cast<__int128>(rows) * hidden;
  const int size = size_of(x_dtype);
  if (overlap({{h_out, n * size}, {codes, n}, {scales, n / group * 4}},
              {{x, n * size}, {residual, n * size}, {weight, static_cast<__int128>(hidden) * size}}))
    return EXLR8_ERR_OVERLAP;
  EXLR8_TIMED(EXLR8_KERNEL_NORM, as_stream(stream),
              launch_residual_rms_q8(x, residual, weight, x_dtype, rows, hidden, group, eps, h_out, codes, scales,
                                     as_stream(stream)));
  return EXLR8_OK;
}

int exlr8_affine4_linear(const void* x, int x_dtype, const float* x_scales, int x_group, int64_t rows,
                         int in_features, int out_features, const uint32_t* codes, const void* scales,
                         const void* biases, int scale_dtype, int group, void* out, int out_dtype, void* stream) {
  const bool q8 = x_dtype == EXLR8_DTYPE_E4M3;
  if ((!valid_act(x_dtype) && !q8) || !valid_act(scale_dtype) || !valid_act(out_dtype)) return EXLR8_ERR_DTYPE;
  if (rows < 0 || rows > (1 << 19) || in_features <= 0 || in_features > (1 << 24) || out_features <= 0 ||
      out_features > (1 << 24))
    return EXLR8_ERR_SHAPE;
  if ((group != 32 && group != 64 && group != 128) || in_features % group) return EXLR8_ERR_SHAPE;
  if (q8 && x_group != in_features &&
      ((x_group != 32 && x_group != 64 && x_group != 128) || in_features % x_group))
    return EXLR8_ERR_SHAPE;
  if (rows == 0) return EXLR8_OK;
  if (!x || !codes || !scales || !out || q8 != (x_scales != nullptr)) return EXLR8_ERR_ARG;
  if (!aligned16(x) || !aligned16(codes)) return EXLR8_ERR_ALIGN;
  const __int128 w = static_cast<__int128>(out_features) * in_features, scale_bytes = w / group * size_of(scale_dtype);
  if (overlap({{out, static_cast<__int128>(rows) * out_features * size_of(out_dtype)}},
              {{x, static_cast<__int128>(rows) * in_features * size_of(x_dtype)},
               {x_scales, q8 ? static_cast<__int128>(rows) * (in_features / x_group) * 4 : 0},
               {codes, w / 2},
               {scales, scale_bytes},
               {biases, scale_bytes}}))
    return EXLR8_ERR_OVERLAP;
  const Affine4Args a{x,     x_dtype, x_scales, q8 ? x_group : in_features, rows, in_features, out_features, codes, scales,
                      biases, scale_dtype, group, out, out_dtype};
  EXLR8_TIMED(EXLR8_KERNEL_LINEAR4, as_stream(stream), launch_affine4_linear(a, as_stream(stream)));
  return EXLR8_OK;
}

int exlr8_latent_append(const void* latent, int64_t latent_stride, const void* rope_key, int64_t rope_stride,
                        int64_t tokens, int rank, int dtype, const void* weight, float eps, const float* cos_sin,
                        int64_t cos_rows, const int32_t* positions, int interleaved, const int64_t* slots, void* cache,
                        int64_t pages, int page_size, const void* q_rope, int64_t q_token_stride, int64_t q_head_stride,
                        int heads, void* q_out, void* stream) {
  if (!half_type(dtype)) return EXLR8_ERR_DTYPE;
  if (tokens < 0 || tokens > kMaxGrid || !rank_ok(rank) || !pages_ok(pages, page_size) || cos_rows < 0)
    return EXLR8_ERR_SHAPE;
  if (q_rope && (heads <= 0 || heads > (1 << 16))) return EXLR8_ERR_SHAPE;
  if (tokens == 0) return EXLR8_OK;
  if (!latent || !rope_key || !slots || (pages > 0 && !cache) || !(eps >= 0.0f) || (cos_sin && !positions) ||
      (q_rope && !q_out))
    return EXLR8_ERR_ARG;
  if (overlap({{cache, static_cast<__int128>(pages) * page_size * (rank + kLatentRope) * 2},
               {q_rope ? q_out : nullptr, static_cast<__int128>(tokens) * heads * kLatentRope * 2}},
              {{latent, tokens, latent_stride, 1, 0, rank},
               {rope_key, tokens, rope_stride, 1, 0, kLatentRope},
               {q_rope, tokens, q_token_stride, heads, q_head_stride, kLatentRope},
               {weight, rank * 2},
               {cos_sin, static_cast<__int128>(cos_rows) * kLatentRope * 4},
               {cos_sin ? positions : nullptr, static_cast<__int128>(tokens) * 4},
               {slots, static_cast<__int128>(tokens) * 8}}))
    return EXLR8_ERR_OVERLAP;
  const LatentAppendArgs a{latent,  latent_stride, rope_key,    rope_stride, tokens, rank,  dtype,
                           weight,  eps,           cos_sin,     cos_rows,    positions, interleaved != 0, slots,
                           cache,   pages * page_size, q_rope,  q_token_stride, q_head_stride, heads, q_out};
  EXLR8_TIMED(EXLR8_KERNEL_APPEND, as_stream(stream), launch_latent_append(a, as_stream(stream)));
  return EXLR8_OK;
}

size_t exlr8_latent_attention_workspace(int64_t batch, int queries, int heads, int rank) {
  if (batch < 0 || batch > (1 << 20) || queries <= 0 || heads <= 0 || heads > (1 << 16) || !rank_ok(rank) ||
      batch * queries * heads > (int64_t{1} << 28))
    return kBadSize;
  return latent_attention_workspace(batch, queries, heads, rank);
}

int exlr8_latent_attention(const void* q_latent, const void* q_rope, int64_t batch, int queries, int heads, int rank,
                           int dtype, const void* cache, int64_t pages, int page_size, const int32_t* block_table,
                           int table_width, const int32_t* lengths, float scale, void* out, float* lse,
                           void* workspace, size_t workspace_bytes, void* stream) {
  if (!half_type(dtype)) return EXLR8_ERR_DTYPE;
  const size_t need = exlr8_latent_attention_workspace(batch, queries, heads, rank);
  if (need == kBadSize || !pages_ok(pages, page_size) || table_width < 0 ||
      static_cast<int64_t>(table_width) * page_size > (1 << 30))
    return EXLR8_ERR_SHAPE;
  if (batch == 0) return EXLR8_OK;
  if (!q_latent || !q_rope || !lengths || !out || (table_width > 0 && !block_table) || (pages > 0 && !cache) ||
      !std::isfinite(scale))
    return EXLR8_ERR_ARG;
  if (!aligned16(q_latent) || !aligned16(q_rope) || !aligned16(cache) || !aligned16(out)) return EXLR8_ERR_ALIGN;
  if (need > 0 && (!workspace || workspace_bytes < need)) return EXLR8_ERR_WORKSPACE;
  if (need > 0 && !aligned16(workspace)) return EXLR8_ERR_ALIGN;
  const __int128 rows = static_cast<__int128>(batch) * queries * heads;
  if (overlap({{out, rows * rank * 2}, {lse, rows * 4}, {workspace, static_cast<__int128>(need)}},
              {{q_latent, rows * rank * 2},
               {q_rope, rows * kLatentRope * 2},
               {cache, static_cast<__int128>(pages) * page_size * (rank + kLatentRope) * 2},
               {block_table, static_cast<__int128>(batch) * table_width * 4},
               {lengths, static_cast<__int128>(batch) * 4}}))
    return EXLR8_ERR_OVERLAP;
  const LatentAttentionArgs a{q_latent,  q_rope,      batch,       queries, heads, rank, dtype, cache, pages,
                              page_size, block_table, table_width, lengths, scale, out,  lse,   workspace};
  EXLR8_TIMED(EXLR8_KERNEL_ATTENTION, as_stream(stream), launch_latent_attention(a, as_stream(stream)));
  return EXLR8_OK;
}

int exlr8_latent_prompt_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                  int64_t k_token_stride, int64_t k_head_stride, const void* k_rope,
                                  int64_t k_rope_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                                  int64_t total_q, int64_t total_k, int heads, int nope, int value, int dtype,
                                  const int32_t* q_starts, const int32_t* k_starts, int seqs, float scale, void* out,
                                  float* lse, void* stream) {
  if (!half_type(dtype)) return EXLR8_ERR_DTYPE;
  if (total_q < 0 || total_k < 0 || total_q > kMaxGrid || total_k > kMaxGrid || heads <= 0 || heads > 65535 ||
      (nope != 64 && nope != 128 && nope != 192) || (value != 64 && value != 128 && value != 192 && value != 256) ||
      seqs < 1 || seqs > 4096)
    return EXLR8_ERR_SHAPE;
  for (const int64_t stride : {q_token_stride, q_head_stride, k_token_stride, k_head_stride, k_rope_stride,
                               v_token_stride, v_head_stride})
    if (stride < 0 || stride % 8 || stride >= (int64_t{1} << 38)) return EXLR8_ERR_SHAPE;
  // Broadcast rows have no tile of their own; a grid holds 2^31 CTAs.
  if ((heads > 1 && (!q_head_stride || !k_head_stride || !v_head_stride)) || (total_q > 1 && !q_token_stride) ||
      (total_k > 1 && (!k_token_stride || !k_rope_stride || !v_token_stride)))
    return EXLR8_ERR_SHAPE;
  if (((total_q + 255) / 256 + seqs) * heads * 2 > kMaxGrid) return EXLR8_ERR_SHAPE;
  if (total_q == 0) return EXLR8_OK;
  if (!q || !out || !q_starts || !k_starts || (total_k > 0 && (!k || !k_rope || !v)) || !std::isfinite(scale))
    return EXLR8_ERR_ARG;
  if (!aligned16(q) || !aligned16(k) || !aligned16(k_rope) || !aligned16(v) || !aligned16(out)) return EXLR8_ERR_ALIGN;
  const __int128 results = static_cast<__int128>(total_q) * heads, starts = 4 * (static_cast<__int128>(seqs) + 1);
  if (overlap({{out, results * value * 2}, {lse, results * 4}},
              {{q, total_q, q_token_stride, heads, q_head_stride, nope + kLatentRope},
               {k, total_k, k_token_stride, heads, k_head_stride, nope},
               {k_rope, total_k, k_rope_stride, 1, 0, kLatentRope},
               {v, total_k, v_token_stride, heads, v_head_stride, value},
               {q_starts, starts},
               {k_starts, starts}}))
    return EXLR8_ERR_OVERLAP;
  const LatentPromptArgs a{q,       k,       k_rope, v,     q_token_stride, q_head_stride, k_token_stride,
                           k_head_stride, k_rope_stride, v_token_stride, v_head_stride, total_q, total_k, heads,
                           nope,    value,   dtype,  q_starts, k_starts, seqs, scale, out, lse};
  EXLR8_TIMED(EXLR8_KERNEL_ATTENTION, as_stream(stream), launch_latent_prompt(a, as_stream(stream)));
  return EXLR8_OK;
}

}  // extern "C"
