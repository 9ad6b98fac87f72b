// y[t][o] = sum_g s[o][g] * sum_{k in g} q[o][k] x[t][k] + b[o][g] * sum_{k in g} x[t][k]
// over 4-bit codes q (eight per uint32, low nibble first), group scales s and
// biases b (b = -8 s without them).
//
// Decoding reads every code once for a handful of rows, so the kernel is
// built to stream.  A CTA takes 128 weight rows in stages of 128 channels (the
// rows' 64 bytes and the channels of x, tensor-map boxes), and two CTAs per SM
// keep their rings full; eight warps multiply with mma.sync m16n8k16 (weights
// on the M side, up to 8 rows of x on the N side; the products need a few
// percent of even the warp-level tensor rate, so tcgen05 would gain nothing,
// and its operands would have to be unpacked through shared memory).  What
// bounds such a kernel after the loads is the integer pipe that unpacks the
// codes, so a code is only masked where it lies.  With float16 products (float16
// x and E4M3 x, which float16 holds exactly) it is the subnormal q 2^-24 or, four
// bits up, q 2^-20: exact, two accumulators.  bfloat16 products would leave
// such sums below float32's normal range, so there a shift and a three-input
// logic operation a pair make it v = 1 + q / 16.  Then, for every unit u of one
// weight scale (and one scale of x),
//   float16:   y = sum_u s_u * (sum_{k in u} q_k x_k) + b_u * (sum_{k in u} x_k)
//   bfloat16:  y = sum_u 16 s_u * (sum_{k in u} v_k x_k)
//                  + (b_u - 16 s_u) * (sum_{k in u} x_k)
// (b = -8 s without biases).  Products are exact and sums float32.  The two terms
// cancel: their rounding is that of sums of |s| (16 + q) |x| and |b - 16 s| |x|
// (float16: of |s| q |x| and |b| |x|), which for weights near zero, codes of 7 to 9
// without biases, are some 70 times the result's own terms |q - 8| |s| |x|; a
// 16-bit output does not show it.  The second sum is a product with ones, which
// lands it in the accumulator's layout.
//
// A warp takes 64 rows (32 when x has more than eight) of a stage; lane t of a
// quad takes word 4 j + t of a row's 16, so that place j is 32 channels: units
// of 32, 64 and 128 are whole places.  The swizzles (64 bytes for the codes, 128
// for x) make both reads free of bank conflicts but for a factor of two on x.
// Float32 x is cut into three bfloat16 pieces that sum to it; scales of E4M3
// codes multiply the unit's sum.  Groups of warps that cover the 128 rows take
// stages in turn, each group in places of its own (a group that waited on
// another's place could be a round ahead of it, and a barrier's parity does not
// tell two rounds apart); the last warp to leave a place has its next stage
// fetched.  The scales come through shared memory too, four stages at a
// time, converted once and laid out a block ahead in three buffers, so that no
// warp waits for more than the others' last block: read by every lane from
// global memory, each load touched eight lines, and groups of 32 took four
// times as long as groups of 128.  (Eight stages at a time: 8 x 6144 x 36864 3%
// faster, 1 x 16384 x 6144 5% slower.)  A cluster of up to eight CTAs shares the
// channels of one row tile where the row tiles alone would not fill the SMs
// evenly; sums are added in a fixed order: the same bits every run.
//
// On the device: 1 row of 16384 x 6144 (50 MB) 23.0 us, 2.3 TB/s; 8 E4M3 rows of
// 6144 x 36864 (113 MB) 30.2 us, 3.9 TB/s; 1 row of 6144 x 576 6.5 us.  The
// schedulers issue in 54% of the cycles with 3.6 warps each, the integer pipe
// is half busy: latency between the two, and the uneven last round of CTAs.

#include <cuda.h>

#include "affine4.cuh"
#include "common.cuh"
#include "launch.cuh"
#include "tensor_map.cuh"
#include "umma.cuh"

namespace exlr8 {

namespace {

constexpr int kRows = 128;   // weight rows of a CTA
constexpr int kChunk = 128;  // channels of a stage
constexpr int kThreads = 256;
constexpr uint32_t kCodeBytes = kRows * 64;
constexpr uint32_t kShared = 104 * 1024;  // two CTAs fit an SM
constexpr int kBlock = 4;                 // stages whose scales are laid out together
constexpr int kMaxStages = 16;

enum XType { kXF32 = EXLR8_DTYPE_F32, kXF16 = EXLR8_DTYPE_F16, kXBF16 = EXLR8_DTYPE_BF16, kXE4M3 = EXLR8_DTYPE_E4M3 };

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool f16) {
  if (f16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Codes i and i + 4 of a word in two 16-bit floats.  bfloat16: 1 + q / 16, q at
// mantissa bits 3 to 6.  float16: the code alone, a subnormal q 2^-24 (even i) or
// q 2^-20 (odd i) where it lies, after one shift for i of 2 and 3.  The mask and
// the ones come in registers: as constants they made two instructions of (v &
// mask) | ones.
template <bool kHalf>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int i, uint32_t mask, uint32_t ones) {
  if (kHalf) return (i < 2 ? w : w >> 8) & (i & 1 ? 0x00F000F0u : 0x000F000Fu);
  const int up = 3 - 4 * i;
  const uint32_t v = up >= 0 ? w << up : w >> -up;
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(ones));
  return r;
}

template <int kX>
constexpr int kXBytes = kX == kXF32 ? 4 : kX == kXE4M3 ? 1 : 2;

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

// Word q (0 to 15) of a token's 128 channels: boxes of 128 bytes a token, 16-byte
// pieces swizzled by the token.
template <int kX, int kTokens>
__device__ __forceinline__ Pieces<kX> load_pieces(const uint8_t* x, int token, int q) {
  Pieces<kX> p;
  const uint8_t* row = x + token * 128;
  if constexpr (kX == kXF32) {
    float f[8];
    row += (q >> 2) * (kTokens * 128);
    const float4 lo = *reinterpret_cast<const float4*>(row + (((q & 3) * 2) ^ (token & 7)) * 16);
    const float4 hi = *reinterpret_cast<const float4*>(row + (((q & 3) * 2 + 1) ^ (token & 7)) * 16);
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
    const uint2 c = *reinterpret_cast<const uint2*>(row + ((q >> 1) ^ (token & 7)) * 16 + (q & 1) * 8);
    const uint32_t even = __byte_perm(c.x, c.y, 0x5140), odd = __byte_perm(c.x, c.y, 0x7362);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t two = static_cast<uint16_t>((i < 2 ? even : odd) >> (16 * (i & 1)));
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(p.v[0][i]) : "h"(two));
    }
  } else {
    row += (q >> 3) * (kTokens * 128);
    const uint4 c = *reinterpret_cast<const uint4*>(row + ((q & 7) ^ (token & 7)) * 16);
    interleave(p.v[0], c.x, c.y, c.z, c.w);
  }
  return p;
}

// What the two sums of a unit count, from the scale and the bias.
template <bool kHalf>
__device__ __forceinline__ float2 scale_pair(float s, float b) {
  return kHalf ? make_float2(16777216.0f * s, b) : make_float2(16.0f * s, fmaf(-16.0f, s, b));
}

// A float at the same shared-memory place of CTA `rank` of the cluster.
__device__ __forceinline__ float load_cluster(const float* p, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(smem_u32(p), rank)));
  return v;
}

// `count` 16-bit values, four at a time where they lie on 8 bytes.
template <int kN>
__device__ __forceinline__ void read16(const uint16_t* p, int count, uint32_t (&v)[kN]) {
  if (kN >= 4 && count == kN && (reinterpret_cast<uintptr_t>(p) & 7) == 0) {
#pragma unroll
    for (int e = 0; e + 3 < kN; e += 4) {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(p + e));
      v[e] = u.x & 0xffffu, v[e + 1] = u.x >> 16, v[e + 2] = u.y & 0xffffu, v[e + 3] = u.y >> 16;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < kN; ++e)
    if (e < count) v[e] = __ldg(p + e);
}

struct Maps {
  CUtensorMap codes, x;
};

template <int kX, int kUnit, int kTiles>
struct Stage {
  static constexpr int kTokens = 8 * kTiles;
  static constexpr int kBoxes = kXBytes<kX>;  // of 128 bytes a token
  static constexpr uint32_t kBytes = kCodeBytes + kBoxes * kTokens * 128;
  static constexpr int kM = kTiles == 1 ? 4 : 2;  // tiles of 16 rows a warp takes
  static constexpr int kWarps = kRows / (16 * kM), kGroups = 8 / kWarps;
  static constexpr int kScales = kBlock * kChunk / kUnit;  // of a row in a block
  // Small units keep a scale and its bias as they are stored, in one word (float32
  // ones are then read where they are used): converted, they would take the
  // ring's place.
  static constexpr bool kPacked = kUnit == 32;
  static constexpr uint32_t kScaleBytes = kScales * kRows * (kPacked ? 4 : 8),
                            kXScaleBytes = kX == kXE4M3 ? kScales * kTokens * 4 : 0;
  static constexpr uint32_t kTail = (3 * (kScaleBytes + kXScaleBytes) + 1023) / 1024 * 1024;
  // Float32 x takes the space of one CTA per SM.
  static constexpr uint32_t kRoom = (kX == kXF32 ? 160 * 1024 : kShared) - kTail;
  static constexpr int kFit = static_cast<int>(kRoom / kBytes / kGroups);
  static constexpr int kDepth = kFit < kMaxStages / kGroups ? kFit : kMaxStages / kGroups;  // places of a group
  static constexpr int kCount = kDepth * kGroups;
  static constexpr int kOutputs = kRows * kTokens;
  static_assert(kDepth >= 2, "one stage is read while the next one lands");
  static_assert(kGroups * kOutputs * 4 <= kCount * kBytes, "the groups' sums lie over the ring");
};

// kUnit: channels that share a weight scale and a scale of x; kTiles: tiles of
// eight rows of x.
template <int kX, int kUnit, int kTiles>
__global__ void __launch_bounds__(kThreads, 2)
    affine4_kernel(const __grid_constant__ Maps maps, const Affine4Args a, int group_shift, int x_shift, int box_rows) {
  using S = Stage<kX, kUnit, kTiles>;
  constexpr bool kHalf = kX == kXF16 || kX == kXE4M3;
  constexpr int kSets = Pieces<kX>::kSets, kM = S::kM;
  constexpr int kUnits = kChunk / kUnit, kPlaces = kUnit / 32;  // units of a stage, places of a unit
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kMaxStages], laid[3];
  __shared__ uint32_t left[kMaxStages];  // warps that have left a place, since the start
  __shared__ float s_sum[S::kOutputs];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int share = blockIdx.z, shares = gridDim.z;  // of the channels; a cluster
  const int o0 = blockIdx.x * kRows;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * S::kTokens;
  const int in = a.in_features;
  const int chunks = (in + kChunk - 1) / kChunk;
  const int begin = static_cast<int>(static_cast<int64_t>(chunks) * share / shares);
  const int stages = static_cast<int>(static_cast<int64_t>(chunks) * (share + 1) / shares) - begin;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kCount; ++i) {
      mbar_init(&full[i], 1);
      left[i] = 0;
    }
    for (int i = 0; i < 3; ++i) mbar_init(&laid[i], 8);
    mbar_fence_init();
  }
  // Rows of x past the box stay zero.
  if (box_rows < S::kTokens) {
    constexpr int kPieces = (S::kBytes - kCodeBytes) / 16;
    for (int i = threadIdx.x; i < S::kCount * kPieces; i += kThreads)
      *reinterpret_cast<uint4*>(smem + i / kPieces * S::kBytes + kCodeBytes + i % kPieces * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_async_smem();
  __syncthreads();
  pdl_wait();
  const int g = lane >> 2, t = lane & 3;
  const int group = warp / S::kWarps;
  // Stage i into its place; one thread.
  auto load = [&](int i, int slot) {
    uint8_t* st = smem + slot * S::kBytes;
    mbar_arrive_expect_tx(&full[slot], kCodeBytes + S::kBoxes * box_rows * 128);
    tma_load_2d(st, &maps.codes, (begin + i) * 16, o0, &full[slot]);
#pragma unroll
    for (int b = 0; b < S::kBoxes; ++b)
      tma_load_2d(st + kCodeBytes + b * (S::kTokens * 128), &maps.x, (begin + i) * kChunk + b * (128 / kXBytes<kX>),
                  static_cast<int>(row0), &full[slot]);
  };
  uint32_t mask, one;
  asm volatile("mov.b32 %0, %1;" : "=r"(mask) : "n"(0x00780078));
  asm volatile("mov.b32 %0, %1;" : "=r"(one) : "n"(kHalf ? 0x3C003C00 : 0x3F803F80));
  // A warp is done with stage i: the last of its group fetches the place's next
  // stage (none waits for another here).
  bool ok = true;
  auto leave = [&](int i, int slot) {
    if (!ok || i + S::kCount >= stages) return;
    uint32_t before;
    asm volatile("atom.acq_rel.cta.shared::cta.add.u32 %0, [%1], 1;"
                 : "=r"(before)
                 : "r"(smem_u32(&left[slot]))
                 : "memory");
    if (before % S::kWarps == S::kWarps - 1) load(i + S::kCount, slot);
  };
  // Stage i belongs to group i % kGroups; its n-th stage to that group's place n % kDepth.
  if (threadIdx.x == 0)
    for (int i = 0; i < min(stages, S::kCount); ++i) load(i, i % S::kGroups * S::kDepth + i / S::kGroups);
  __syncwarp();
  float out[kTiles][kM][4];
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) out[n][m][e] = 0.0f;
  const int r0 = 16 * kM * (warp % S::kWarps) + g;  // the first of the lane's rows, eight apart
  // Scales of a block: thread (row, half of the block's groups) reads them raw,
  // two blocks ahead, and leaves 16 s and b - 16 s; rows past the last are the
  // last again (their results are not stored).
  uint32_t* const s_raw = reinterpret_cast<uint32_t*>(smem + S::kCount * S::kBytes);
  float2* const s_scale = reinterpret_cast<float2*>(smem + S::kCount * S::kBytes);  // [3][kScales][kRows]
  float* const s_x = reinterpret_cast<float*>(smem + S::kCount * S::kBytes + 3 * S::kScaleBytes);  // [3][kScales][kTokens]
  const int groups = in >> group_shift;
  const int per = (kBlock * kChunk >> group_shift) / 2;  // groups a thread reads of a block
  const int scale_row = threadIdx.x % kRows, scale_half = threadIdx.x / kRows;
  const int64_t scale_at = static_cast<int64_t>(min(o0 + scale_row, a.out_features - 1)) * groups;
  constexpr int kPer = S::kScales / 2;
  uint32_t raw_s[kPer], raw_b[kPer];
  float raw_x = 0.0f;
  auto fetch = [&](int block) {
    const int first = ((begin + block * kBlock) * kChunk >> group_shift) + scale_half * per;
#pragma unroll
    for (int e = 0; e < kPer; ++e) raw_s[e] = raw_b[e] = 0;
    if (a.scale_dtype == kF32) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if (S::kPacked || e >= per || first + e >= groups) continue;
        raw_s[e] = __ldg(static_cast<const uint32_t*>(a.scales) + scale_at + first + e);
        if (a.biases) raw_b[e] = __ldg(static_cast<const uint32_t*>(a.biases) + scale_at + first + e);
      }
    } else {
      read16(static_cast<const uint16_t*>(a.scales) + scale_at + first, min(per, groups - first), raw_s);
      if (a.biases) read16(static_cast<const uint16_t*>(a.biases) + scale_at + first, min(per, groups - first), raw_b);
    }
    if (kX == kXE4M3 && threadIdx.x < S::kScales * S::kTokens) {
      const int k0 = (begin + block * kBlock) * kChunk + threadIdx.x / S::kTokens * kUnit;
      const int64_t token = row0 + threadIdx.x % S::kTokens;
      raw_x = token < a.rows && k0 < in
                  ? __ldg(a.x_scales + (a.x_group == in ? token : token * (in >> x_shift) + (k0 >> x_shift)))
                  : 0.0f;
    }
  };
  auto lay = [&](int buffer) {
    if (S::kPacked) {
      uint32_t* dst = s_raw + buffer * S::kScales * kRows + scale_half * per * kRows + scale_row;
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (e < per) dst[e * kRows] = raw_s[e] | raw_b[e] << 16;
    } else {
      float2* dst = s_scale + buffer * S::kScales * kRows + scale_half * per * kRows + scale_row;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if (e >= per) continue;
        float v = __uint_as_float(raw_s[e]), b = __uint_as_float(raw_b[e]);
        if (a.scale_dtype == kBF16) {
          v = __uint_as_float(raw_s[e] << 16);
          b = __uint_as_float(raw_b[e] << 16);
        } else if (a.scale_dtype == kF16) {
          v = __half2float(__ushort_as_half(static_cast<unsigned short>(raw_s[e])));
          b = __half2float(__ushort_as_half(static_cast<unsigned short>(raw_b[e])));
        }
        dst[e * kRows] = scale_pair<kHalf>(v, a.biases ? b : -8.0f * v);
      }
    }
    if (kX == kXE4M3 && threadIdx.x < S::kScales * S::kTokens)
      s_x[buffer * S::kScales * S::kTokens + threadIdx.x] = raw_x;
    __syncwarp();
    if (lane == 0) mbar_arrive(&laid[buffer]);
  };
  const int blocks = (stages + kBlock - 1) / kBlock;
  fetch(0);
  lay(0);
  if (blocks > 1) fetch(1);
  int slot = group * S::kDepth, buffer = 0;
  uint32_t round = 0, lap = 0;
  for (int block = 0; block < blocks; ++block) {
    // Every warp has laid its part of this block, so none is still at the block
    // before the last, whose buffer takes the next one.
    ok = ok && mbar_wait(&laid[buffer], lap);
    if (block + 1 < blocks) lay(buffer == 2 ? 0 : buffer + 1);
    if (block + 2 < blocks) fetch(block + 2);
    for (int i = block * kBlock + group; i < min(stages, (block + 1) * kBlock); i += S::kGroups) {
      ok = ok && mbar_wait(&full[slot], round);
      const uint8_t* st = smem + slot * S::kBytes;
      // Word 4 j + t of row r0 + 8 r: 16-byte piece j of the row's four, swizzled
      // by bits 1 and 2 of the row.
      const uint8_t* w0 = st + r0 * 64 + t * 4;
      const int swizzle = (g >> 1) & 3;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (kUnits > 1 && (begin + i) * kChunk + u * kUnit >= in) break;
        // [0]: the sums of codes i = 0 and 2, [1]: of 1 and 3 (float16), else of all.
        float acc[kHalf ? 2 : 1][kTiles][kM][4] = {}, ones[kTiles][4] = {};
#pragma unroll
        for (int j = u * kPlaces; j < (u + 1) * kPlaces; ++j) {
          uint32_t w[2 * kM];
#pragma unroll
          for (int r = 0; r < 2 * kM; ++r) w[r] = *reinterpret_cast<const uint32_t*>(w0 + r * 512 + ((j ^ swizzle) << 4));
          Pieces<kX> x[kTiles];
#pragma unroll
          for (int n = 0; n < kTiles; ++n) x[n] = load_pieces<kX, S::kTokens>(st + kCodeBytes, 8 * n + g, 4 * j + t);
#pragma unroll
          for (int p = 0; p < 2; ++p) {
#pragma unroll
            for (int m = 0; m < kM; ++m) {
              const int i0 = kHalf ? p : 2 * p, i1 = kHalf ? p + 2 : 2 * p + 1;
              const uint32_t av[4] = {code_pair<kHalf>(w[2 * m], i0, mask, one),
                                      code_pair<kHalf>(w[2 * m + 1], i0, mask, one),
                                      code_pair<kHalf>(w[2 * m], i1, mask, one),
                                      code_pair<kHalf>(w[2 * m + 1], i1, mask, one)};
#pragma unroll
              for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int set = 0; set < kSets; ++set)
                  mma(acc[kHalf ? p : 0][n][m], av, x[n].v[set][i0], x[n].v[set][i1], kHalf);
            }
            const uint32_t av[4] = {one, one, one, one};
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
              for (int set = 0; set < kSets; ++set) mma(ones[n], av, x[n].v[set][2 * p], x[n].v[set][2 * p + 1], kHalf);
          }
        }
        if (u == kUnits - 1) {
          __syncwarp();
          if (lane == 0) leave(i, slot);
        }
        const int at = (i % kBlock) * kChunk + u * kUnit;  // channel in the block
        const float2* scale = s_scale + (buffer * S::kScales + (at >> group_shift)) * kRows + r0;
        float xs[kTiles][2];
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int f = 0; f < 2; ++f)
            xs[n][f] = kX == kXE4M3 ? s_x[(buffer * S::kScales + at / kUnit) * S::kTokens + 8 * n + 2 * t + f] : 1.0f;
#pragma unroll
        for (int r = 0; r < 2 * kM; ++r) {
          float2 v;
          if (S::kPacked) {
            if (a.scale_dtype == kF32) {
              const int64_t from = static_cast<int64_t>(min(o0 + r0 + 8 * r, a.out_features - 1)) * groups +
                                   (((begin + i) * kChunk + u * kUnit) >> group_shift);
              v.x = __ldg(static_cast<const float*>(a.scales) + from);
              v.y = a.biases ? __ldg(static_cast<const float*>(a.biases) + from) : 0.0f;
            } else {
              const uint32_t raw = s_raw[(buffer * S::kScales + (at >> group_shift)) * kRows + r0 + 8 * r];
              v = a.scale_dtype == kBF16 ? make_float2(__uint_as_float(raw << 16), __uint_as_float(raw & 0xffff0000u))
                                         : __half22float2(*reinterpret_cast<const __half2*>(&raw));
            }
            v = scale_pair<kHalf>(v.x, a.biases ? v.y : -8.0f * v.x);
          } else {
            v = scale[8 * r];
          }
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
              float& o = out[n][r / 2][2 * (r & 1) + f];
              float sum = acc[0][n][r / 2][2 * (r & 1) + f];
              if (kHalf) sum = fmaf(acc[kHalf][n][r / 2][2 * (r & 1) + f], 0.0625f, sum);
              const float y = fmaf(ones[n][f], v.y, sum * v.x);
              o = kX == kXE4M3 ? fmaf(y, xs[n][f], o) : o + y;
            }
        }
      }
      __syncwarp();
      if (++slot == (group + 1) * S::kDepth) {
        slot = group * S::kDepth;
        round ^= 1;
      }
    }
    if (++buffer == 3) {
      buffer = 0;
      lap ^= 1;
    }
  }
  // Accumulator e of a lane is row r0 + 16 m + 8 (e / 2), token 8 n + 2 t + e % 2.
  auto place = [&](int n, int m, int e) { return (8 * n + 2 * t + (e & 1)) * kRows + r0 + 16 * m + 8 * (e >> 1); };
  // Where a wait ran out, copies still in flight land before the memory goes on.
  if (!__syncthreads_and(ok)) {
    ok = false;
    if (threadIdx.x == 0)
      for (int u = max(0, stages - S::kCount); u < stages; ++u)
        mbar_wait(&full[u % S::kGroups * S::kDepth + u / S::kGroups % S::kDepth], (u / S::kCount) & 1);
    __syncthreads();
  }
  float* sums = reinterpret_cast<float*>(smem);  // over the ring, which every warp has left
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[group * S::kOutputs + place(n, m, e)] = ok ? out[n][m][e] : NAN;
  __syncthreads();
  for (int i = threadIdx.x; i < S::kOutputs; i += kThreads) {
    float v = sums[i];
#pragma unroll
    for (int r = 1; r < S::kGroups; ++r) v += sums[r * S::kOutputs + i];
    s_sum[i] = v;
  }
  // (a cluster's barrier wants whole warps)
  __syncwarp();
  if (shares > 1) cluster_sync();
  else __syncthreads();
  for (int i = share * kThreads + threadIdx.x; i < S::kOutputs; i += shares * kThreads) {
    const int o = o0 + i % kRows;
    const int64_t token = row0 + i / kRows;
    if (o >= a.out_features || token >= a.rows) continue;
    float v = shares > 1 ? load_cluster(&s_sum[i], 0) : s_sum[i];
    for (int r = 1; r < shares; ++r) v += load_cluster(&s_sum[i], r);
    store_act(a.out, a.out_dtype, token * a.out_features + o, v);
  }
  __syncwarp();  // (some lanes stored, others had no row)
  if (shares > 1) cluster_sync();  // no CTA of the cluster leaves while its sums are read
}

int log2_of(int v) {
  int n = 0;
  while ((1 << n) < v) ++n;
  return n;
}

// CTAs that share a row tile's channels: the count with the fewest rounds per
// share, at least four stages each.  A cluster lies within one GPC (eight of 16
// to 20 SMs, two CTAs per SM), so clusters of six fill less of the GPU than
// those of five: 48 row tiles of 16384 channels took 27 us by five, 37 by six.
int channel_shares(int64_t tiles, int chunks, int sms) {
  int best = 1;
  double least = 1e30;
  for (int n = 1; n <= 8 && (n == 1 || chunks >= 4 * n); ++n) {
    const int64_t fit = n == 1 ? 2 * sms : sms / 18 * (32 / n), rounds = (tiles + fit - 1) / fit;
    const double cost = static_cast<double>(rounds) / n + 0.01 * n;
    if (cost < least) {
      least = cost;
      best = n;
    }
  }
  return best;
}

template <int kX, int kUnit, int kTiles>
cudaError_t launch(const Affine4Args& a, cudaStream_t s) {
  using S = Stage<kX, kUnit, kTiles>;
  int device = 0, sms = 148;
  if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  const int box_rows = static_cast<int>(a.rows < S::kTokens ? a.rows : S::kTokens);
  const CUtensorMapDataType type = kX == kXF32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : kX == kXE4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : kX == kXF16  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  Maps maps;
  const uint64_t in = static_cast<uint64_t>(a.in_features);
  if (!encode_tiled_2d(&maps.codes, CU_TENSOR_MAP_DATA_TYPE_UINT32, a.codes, in / 8, a.out_features, in / 2, 16, kRows,
                       CU_TENSOR_MAP_SWIZZLE_64B) ||
      !encode_tiled_2d(&maps.x, type, a.x, in, a.rows, in * kXBytes<kX>, 128 / kXBytes<kX>, box_rows,
                       CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  auto kernel = affine4_kernel<kX, kUnit, kTiles>;
  constexpr int kBytes = S::kCount * S::kBytes + S::kTail + 1024;
  static std::atomic<uint64_t> ready{0};
  cudaError_t err = allow_shared_memory(kernel, kBytes, ready);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((a.out_features + kRows - 1) / kRows, static_cast<unsigned>((a.rows + S::kTokens - 1) / S::kTokens));
  cfg.gridDim.z = channel_shares(static_cast<int64_t>(cfg.gridDim.x) * cfg.gridDim.y, (a.in_features + kChunk - 1) / kChunk,
                                 sms);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = cfg.gridDim.z;
  cfg.attrs = attr;
  cfg.numAttrs = cfg.gridDim.z > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, maps, a, log2_of(a.group),
                            kX == kXE4M3 && a.x_group != a.in_features ? log2_of(a.x_group) : 0, box_rows);
}

template <int kX, int kUnit>
cudaError_t launch_tiles(const Affine4Args& a, cudaStream_t s) {
  return a.rows <= 8 ? launch<kX, kUnit, 1>(a, s) : launch<kX, kUnit, 2>(a, s);
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
