// y[t][o] = sum_g s[o][g] * sum_{k in g} q[o][k] x[t][k] + b[o][g] * sum_{k in g} x[t][k]
// over 4-bit codes q (eight per uint32, low nibble first), group scales s and
// biases b (b = -8 s without them).
//
// Decoding reads every code once for a handful of rows, so the kernel is
// built to stream: each warp loads 32 weight rows x 128 or 256 channels as 16-byte
// pieces straight into registers, one iteration ahead, and multiplies them
// with mma.sync m16n8k16 (weights on the M side, up to 8 rows of x on the N
// side; the products need a few percent of even the warp-level tensor rate, so
// nothing is gained from tcgen05, whose operands would have to pass through
// shared memory first).  A code becomes the 16-bit float q - 8 exactly: the
// nibble is or-ed into the mantissa of 128 (bfloat16) or 1024 (float16) and
// 136 or 1032 subtracted.  Products are exact, sums are float32:
//   y = sum_u s_u * (sum_{k in u} (q_k - 8) x_k) + (b_u + 8 s_u) * (sum_{k in u} x_k)
// for every unit u of one weight scale (and one scale of x).  The second sum
// is a product with ones, which lands it in the accumulator's layout.
//
// A lane's 16 bytes are 32 channels of one row, while a unit of 32 or 64
// channels has to meet in one instruction across the four lanes of a quad:
// one or two shuffle exchanges inside the quad re-deal the words, and x is
// read in the dealt order.  Float32 x is cut into three bfloat16 pieces that
// sum to it; E4M3 codes are exact in float16 and their scales multiply the
// unit's sum.  The warps of a CTA take the channels in turn and add their
// results in shared memory in warp order: the same bits every run.

#include "affine4.cuh"
#include "common.cuh"
#include "launch.cuh"

namespace exlr8 {

namespace {

constexpr int kRows = 32;    // weight rows of a CTA
constexpr int kChunk = 128;  // channels of one dealt set of words

enum XType { kXF32 = EXLR8_DTYPE_F32, kXF16 = EXLR8_DTYPE_F16, kXBF16 = EXLR8_DTYPE_BF16, kXE4M3 = EXLR8_DTYPE_E4M3 };

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool f16) {
  if (f16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Codes i and i + 4 of a word as two 16-bit floats, minus 8.
template <bool kHalf>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int i) {
  const uint32_t v = ((w >> (4 * i)) & 0x000F000Fu) | (kHalf ? 0x64006400u : 0x43004300u);
  uint32_t r;
  if (kHalf) asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x64086408u));
  else asm("sub.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x43084308u));
  return r;
}

__device__ __forceinline__ uint4 load_codes(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Eight channels of x as up to three sets of the four words (x0, x4), (x1,
// x5), (x2, x6), (x3, x7).
template <int kX>
struct Pieces {
  static constexpr int kSets = kX == kXF32 ? 3 : 1;
  uint32_t v[kSets][4];
};

__device__ __forceinline__ void interleave(uint32_t (&v)[4], uint32_t x01, uint32_t x23, uint32_t x45, uint32_t x67) {
  v[0] = __byte_perm(x01, x45, 0x5410);
  v[1] = __byte_perm(x01, x45, 0x7632);
  v[2] = __byte_perm(x23, x67, 0x5410);
  v[3] = __byte_perm(x23, x67, 0x7632);
}

template <int kX>
__device__ __forceinline__ Pieces<kX> load_pieces(const void* x, int64_t at, bool there) {
  Pieces<kX> p;
  if constexpr (kX == kXF32) {
    float f[8];
    const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(x) + at);
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 lo = there ? __ldg(src) : zero, hi = there ? __ldg(src + 1) : zero;
    f[0] = lo.x, f[1] = lo.y, f[2] = lo.z, f[3] = lo.w, f[4] = hi.x, f[5] = hi.y, f[6] = hi.z, f[7] = hi.w;
#pragma unroll
    for (int s = 0; s < 3; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p.v[s][i]) : "f"(f[i + 4]), "f"(f[i]));
        // An infinite or NaN first piece is the value; its remainder is not.
        const float r0 = f[i] - __uint_as_float(p.v[s][i] << 16), r1 = f[i + 4] - __uint_as_float(p.v[s][i] & 0xffff0000u);
        f[i] = s == 0 && !(fabsf(f[i]) < INFINITY) ? 0.0f : r0;
        f[i + 4] = s == 0 && !(fabsf(f[i + 4]) < INFINITY) ? 0.0f : r1;
      }
  } else if constexpr (kX == kXE4M3) {
    const uint2 c = there ? __ldg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(x) + at)) : make_uint2(0, 0);
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t two = static_cast<uint16_t>((i < 2 ? c.x : c.y) >> (16 * (i & 1)));
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[i]) : "h"(two));
    }
    interleave(p.v[0], h[0], h[1], h[2], h[3]);
  } else {
    const uint4 c = there ? __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + at))
                          : make_uint4(0, 0, 0, 0);
    interleave(p.v[0], c.x, c.y, c.z, c.w);
  }
  return p;
}

// Re-deal a lane's four words so that the words of one unit lie in one place
// of all four lanes of the quad.
template <int kUnit>
__device__ __forceinline__ void deal(uint4& w, int t) {
  if constexpr (kUnit <= 64) {
    const bool low = t < 2;
    uint32_t a = low ? w.z : w.x, b = low ? w.w : w.y;
    a = __shfl_xor_sync(0xffffffffu, a, 2);
    b = __shfl_xor_sync(0xffffffffu, b, 2);
    w = low ? make_uint4(w.x, w.y, a, b) : make_uint4(a, b, w.z, w.w);
  }
  if constexpr (kUnit <= 32) {
    const bool even = (t & 1) == 0;
    uint32_t a = even ? w.y : w.x, b = even ? w.w : w.z;
    a = __shfl_xor_sync(0xffffffffu, a, 1);
    b = __shfl_xor_sync(0xffffffffu, b, 1);
    w = even ? make_uint4(w.x, a, w.z, b) : make_uint4(a, w.y, b, w.w);
  }
}

// The word of a chunk that lane t of a quad holds in place j after the deal.
template <int kUnit>
__device__ __forceinline__ int dealt(int t, int j) {
  if (kUnit >= 128) return 4 * t + j;
  if (kUnit == 64) return 8 * (j >> 1) + 4 * (t & 1) + 2 * (t >> 1) + (j & 1);
  return 4 * j + t;
}

// kUnit: channels that share a weight scale and a scale of x; kTiles: tiles of
// eight rows of x.
template <int kX, int kUnit, int kTiles, bool kBias>
__global__ void __launch_bounds__(256, 2) affine4_kernel(const Affine4Args a) {
  constexpr bool kHalf = kX == kXF16 || kX == kXE4M3;
  constexpr int kSets = Pieces<kX>::kSets;
  constexpr int kPlaces = kUnit / 32;  // word places of a unit
  // Chunks an iteration: two keep 128 bytes of a row in one warp; where x takes
  // more registers, one avoids spills.
  constexpr int kDepth = kTiles == 1 && kX != kXF32 ? 2 : 1;
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float s_part[8][kTiles * 2][4][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int o0 = blockIdx.x * kRows;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * (8 * kTiles);
  const int groups = a.in_features / a.group, x_groups = kX == kXE4M3 ? a.in_features / a.x_group : 0;
  const int chunks = (a.in_features + kChunk - 1) / kChunk;
  // Rows past the last are the last again; their results are not stored.
  const uint4* codes[4];
  int64_t scale_row[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int o = min(o0 + 8 * r + g, a.out_features - 1);
    codes[r] = reinterpret_cast<const uint4*>(a.codes + static_cast<int64_t>(o) * (a.in_features / 8)) + t;
    scale_row[r] = static_cast<int64_t>(o) * groups;
  }
  float out[kTiles][2][4];
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) out[n][m][e] = 0.0f;

  // The next iteration's codes are in flight during this one's products.
  uint4 next[kDepth][4];
  auto fetch = [&](int c) {
#pragma unroll
    for (int h = 0; h < kDepth; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        next[h][r] = (c + h) * kChunk + 32 * t < a.in_features ? load_codes(codes[r] + (c + h) * 4)
                                                              : make_uint4(0, 0, 0, 0);
  };
  if (kDepth * warp < chunks) fetch(kDepth * warp);
  for (int c0 = kDepth * warp; c0 < chunks; c0 += 8 * kDepth) {
    uint4 now[kDepth][4];
#pragma unroll
    for (int h = 0; h < kDepth; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) now[h][r] = next[h][r];
    if (c0 + 8 * kDepth < chunks) fetch(c0 + 8 * kDepth);
#pragma unroll
    for (int h = 0; h < kDepth; ++h) {
      const int c = c0 + h;
      if (c >= chunks) break;
#pragma unroll
      for (int r = 0; r < 4; ++r) deal<kUnit>(now[h][r], t);
#pragma unroll
      for (int u = 0; u < kChunk / kUnit; ++u) {
        const int k0 = c * kChunk + u * kUnit;
        if (kUnit < kChunk && k0 >= a.in_features) break;
        float s[4], b[4];
        const int gi = min(k0 / a.group, groups - 1);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[r] = load_act(a.scales, a.scale_dtype, scale_row[r] + gi);
          if (kBias) b[r] = fmaf(8.0f, s[r], load_act(a.biases, a.scale_dtype, scale_row[r] + gi));
        }
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          float acc[2][4] = {}, ones[4] = {};
          const int64_t row = row0 + 8 * n + g;
#pragma unroll
          for (int j = u * kPlaces; j < (u + 1) * kPlaces; ++j) {
            const int k = c * kChunk + 8 * dealt<kUnit>(t, j);
            const Pieces<kX> x =
                load_pieces<kX>(a.x, row * a.in_features + k, row < a.rows && k < a.in_features);
#pragma unroll
            for (int p = 0; p < 2; ++p) {
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                const uint4 &wa = now[h][2 * m], &wb = now[h][2 * m + 1];
                const uint32_t va = j == 0 ? wa.x : j == 1 ? wa.y : j == 2 ? wa.z : wa.w;
                const uint32_t vb = j == 0 ? wb.x : j == 1 ? wb.y : j == 2 ? wb.z : wb.w;
                const uint32_t av[4] = {code_pair<kHalf>(va, 2 * p), code_pair<kHalf>(vb, 2 * p),
                                        code_pair<kHalf>(va, 2 * p + 1), code_pair<kHalf>(vb, 2 * p + 1)};
#pragma unroll
                for (int set = 0; set < kSets; ++set)
                  mma(acc[m], av, x.v[set][2 * p], x.v[set][2 * p + 1], kHalf);
              }
              if (kBias) {
                const uint32_t one = kHalf ? 0x3C003C00u : 0x3F803F80u;
                const uint32_t av[4] = {one, one, one, one};
#pragma unroll
                for (int set = 0; set < kSets; ++set) mma(ones, av, x.v[set][2 * p], x.v[set][2 * p + 1], kHalf);
              }
            }
          }
          float xs[2] = {1.0f, 1.0f};
          if (kX == kXE4M3) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int64_t token = row0 + 8 * n + 2 * t + e;
              if (token < a.rows) xs[e] = __ldg(a.x_scales + token * x_groups + k0 / a.x_group);
            }
          }
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = 2 * m + (e >> 1);
              float v = acc[m][e] * s[r];
              if (kBias) v = fmaf(b[r], ones[e & 1], v);
              if (kX == kXE4M3) out[n][m][e] = fmaf(v, xs[e & 1], out[n][m][e]);
              else out[n][m][e] += v;
            }
        }
      }
    }
  }
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) s_part[warp][2 * n + m][e][lane] = out[n][m][e];
  __syncthreads();
  // Output (row o, token): accumulator e of lane 4 * (o % 8) + token / 2 % 4.
  for (int i = threadIdx.x; i < kRows * 8 * kTiles; i += 256) {
    const int o = i % kRows, token = i / kRows;
    if (o0 + o >= a.out_features || row0 + token >= a.rows) continue;
    const int tile = 2 * (token / 8) + o / 16, e = 2 * (o / 8 & 1) + (token & 1), l = 4 * (o & 7) + (token / 2 & 3);
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += s_part[w][tile][e][l];
    store_act(a.out, a.out_dtype, (row0 + token) * a.out_features + o0 + o, v);
  }
}

template <int kX, int kUnit, int kTiles>
cudaError_t launch_bias(const Affine4Args& a, cudaStream_t s) {
  const dim3 grid((a.out_features + kRows - 1) / kRows, static_cast<unsigned>((a.rows + 8 * kTiles - 1) / (8 * kTiles)));
  if (a.biases) return launch_pdl(affine4_kernel<kX, kUnit, kTiles, true>, grid, dim3(256), 0, s, a);
  return launch_pdl(affine4_kernel<kX, kUnit, kTiles, false>, grid, dim3(256), 0, s, a);
}

template <int kX, int kUnit>
cudaError_t launch_tiles(const Affine4Args& a, cudaStream_t s) {
  return a.rows <= 8 ? launch_bias<kX, kUnit, 1>(a, s) : launch_bias<kX, kUnit, 2>(a, s);
}

template <int kX>
cudaError_t launch_unit(const Affine4Args& a, cudaStream_t s) {
  const int unit = a.x_group < a.group ? a.x_group : a.group;
  if (unit == 32) return launch_tiles<kX, 32>(a, s);
  if (unit == 64) return launch_tiles<kX, 64>(a, s);
  return launch_tiles<kX, 128>(a, s);
}

}  // namespace

cudaError_t launch_affine4_linear(const Affine4Args& a, cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  switch (a.x_dtype) {
    case kXF32: return launch_unit<kXF32>(a, s);
    case kXF16: return launch_unit<kXF16>(a, s);
    case kXBF16: return launch_unit<kXBF16>(a, s);
    default: return launch_unit<kXE4M3>(a, s);
  }
}

}  // namespace exlr8
