// Causal attention of ragged prompts over expanded keys and values: head h of
// key j is [k_j,h, k_rope_j] (the rotary part is shared by all heads) and its
// value v_j,h.  Query i of a sequence with n queries and m keys sees its
// first m - n + 1 + i keys, so a chunk with a history ends with its keys.  A
// query that sees none gives zeros (and lse -inf).
//
// One CTA takes 256 queries of one head, as two tiles of 128 rows, and walks
// the keys in tiles.  For each query tile q and key tile j
//   S_q = Q_q K_j^T                      tcgen05, both operands in shared memory
//   P_q = 2^(c S_q - c m + 6)            one thread per row, float32
//   O_q += P_q V_j                       tcgen05, P_q from tensor memory
// with c = |scale| log2(e) (a negative scale negates Q in the instruction),
// m a running maximum and l = sum P the float32 sum of the unrounded weights.
// m is raised only when a row's maximum has grown by more than 2^8 (then O and
// l are multiplied once and the tile is weighed again), so a tile is weighed
// without a pass for its maximum first, and P stays below 2^14 and float16 weights keep their
// full precision down to 2^-20 of the largest.  Tensor memory is full: S_0,
// S_1, O_0, O_1 of 128 columns each, P_q over S_q.  While the threads of one
// query tile form its weights the tensor pipe works for the other one, which
// is why two tiles share a CTA (and why each K and V tile is read from L2
// once for 256 queries).
//
// The two query tiles leave room for 1.6 tiles of keys and values (at 192 key
// channels), so K and V tiles share one ring of blocks of 64 channels, in the
// order of their use: the next V lands while this one is multiplied, the next
// but one K as soon as it is done.  (Two places for K and one for V left the
// tensor pipe waiting for V in every tile: 757 us for 8192 queries of 32 heads.)
//
// The softmax of a tile adds and multiplies two float32 at a time: issue slots,
// not the special-function unit, bounded it (655 us to 576 us; taking a part of
// the exponentials from a polynomial on the multiply-add pipe gained nothing).
//
// Warp 0 loads (TMA), warp 1 issues the matrix instructions, warps 4-7 and
// 8-11 are the softmax of query tiles 0 and 1 and take registers that the first
// four give up.  Value channels beyond 128 are
// a second CTA's (the scores are formed again there).  Rows of the last key
// tile that belong to no key of the sequence are zeroed in the V tile, since
// 0 x NaN would reach the sum.  Waits are bounded; one that runs out leaves
// NaN in the CTA's output.

#include <cuda.h>

#include "common.cuh"
#include "latent.cuh"
#include "launch.cuh"
#include "tensor_map.cuh"
#include "umma.cuh"

namespace exlr8 {

namespace {

constexpr int kThreads = 384;
// Registers a thread: 168 at launch, then 72 and 208, 128 * 72 + 256 * 208 of
// the 384 * 168 that the block holds.
constexpr int kFewRegisters = 72, kManyRegisters = 208;
static_assert(128 * kFewRegisters + 256 * kManyRegisters <= 384 * 168, "more than the block holds");
constexpr int kTileQ = 128;
constexpr float kLift = 6.0f;       // weights are 2^6 of their share of the maximum
constexpr float kLag = 8.0f;        // log2 by which a maximum may lag
constexpr uint32_t kSmem = 229376;  // 224 KB of operand tiles

template <int kBlocks>  // 64-channel blocks of a key: 2, 3 or 4
struct Tiles {
  static constexpr int kKeys = kBlocks == 4 ? 64 : 128;
  static constexpr uint32_t kQ = kBlocks * 16384;    // one query tile
  static constexpr uint32_t kBlock = kKeys * 128;    // 64 channels of a key or value tile
  static constexpr int kRing = (kSmem - 2 * kQ) / kBlock;
  static_assert(kRing >= kBlocks + 4, "a key tile and two value tiles");
};

constexpr int kUnits = 8;  // key and value tiles that the barriers tell apart; the ring holds five at most

struct Shared {
  uint64_t q_full, full[kUnits], empty[kUnits];
  uint64_t s_full[2], p_ready[2], o_done[2];
  uint32_t tmem;
  int seq, tile;
};

struct Maps {
  CUtensorMap q, k, r, v;
  int q_swap, k_swap, v_swap;  // dimension order (channels, tokens, heads)
};

__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* map, int swap, int channel, int head, int row,
                                          uint64_t* bar) {
  if (swap) tma_load_3d(dst, map, channel, row, head, bar);
  else tma_load_3d(dst, map, channel, head, row, bar);
}

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Two float32 in one register pair: sm_100 adds and multiplies both at once.
__device__ __forceinline__ uint64_t both(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void apart(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <int kAct>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t r;
  if (kAct == kF16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <int kAct, int kBlocks>
__global__ void __launch_bounds__(kThreads, 1)
    latent_prompt_kernel(const __grid_constant__ Maps maps, const LatentPromptArgs a, int value_parts) {
  using T = Tiles<kBlocks>;
  constexpr int kKeys = T::kKeys;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared sh;
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* const ring = smem + 2 * T::kQ;
  const int warp = static_cast<int>(uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const int columns = a.heads * value_parts;
  const int head = blockIdx.x % columns / value_parts, part = blockIdx.x % value_parts;

  // The CTA's sequence and its tile of 256 queries: tiles are numbered over
  // the sequences and taken from the last (its rows see the most keys).
  pdl_launch_dependents();
  pdl_wait();
  auto start_of = [&](const int32_t* starts, int s, int64_t total) {
    return min(max(starts[s], 0), static_cast<int>(total));
  };
  auto tiles_of = [&](int s) {
    const int n = s < a.seqs ? start_of(a.q_starts, s + 1, a.total_q) - start_of(a.q_starts, s, a.total_q) : 0;
    return (max(n, 0) + 255) / 256;
  };
  if (warp == 0) {
    int total = 0;
    for (int s0 = 0; s0 < a.seqs; s0 += 32) total += __reduce_add_sync(0xffffffffu, tiles_of(s0 + lane));
    int at = total - 1 - static_cast<int>(blockIdx.x / columns), found = -1, tile = 0;
    for (int s0 = 0; s0 < a.seqs && at >= 0 && found < 0; s0 += 32) {
      const int n = tiles_of(s0 + lane);
      int end = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, end, off);
        if (lane >= off) end += other;
      }
      const uint32_t mine = __ballot_sync(0xffffffffu, at < end);
      if (mine) {
        const int which = __ffs(mine) - 1;
        tile = at - __shfl_sync(0xffffffffu, end - n, which);
        found = s0 + which;
      } else {
        at -= __shfl_sync(0xffffffffu, end, 31);
      }
    }
    if (lane == 0) {
      sh.seq = found;
      sh.tile = tile;
      mbar_init(&sh.q_full, 1);
      for (int i = 0; i < kUnits; ++i) {
        mbar_init(&sh.full[i], 1);
        mbar_init(&sh.empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sh.s_full[i], 1);
        mbar_init(&sh.p_ready[i], kTileQ);
        mbar_init(&sh.o_done[i], 1);
      }
      mbar_fence_init();
    }
  }
  __syncthreads();
  if (sh.seq < 0) return;
  const int q0 = start_of(a.q_starts, sh.seq, a.total_q);
  const int queries = start_of(a.q_starts, sh.seq + 1, a.total_q) - q0;
  const int k0 = start_of(a.k_starts, sh.seq, a.total_k);
  const int keys = max(start_of(a.k_starts, sh.seq + 1, a.total_k) - k0, 0);
  const int first = sh.tile * 256;
  const int vb = min(2, a.value / 64 - 2 * part);  // 64-channel value blocks of this CTA
  // Key tiles of each query tile: its last query sees the most keys.
  int tiles[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int last = min(first + (q + 1) * kTileQ, queries) - 1;
    const int seen = last >= first + q * kTileQ ? min(keys - queries + 1 + last, keys) : 0;
    tiles[q] = seen > 0 ? (seen + kKeys - 1) / kKeys : 0;
  }
  const int all = max(tiles[0], tiles[1]);
  if (warp == 1) tmem_alloc(&sh.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
    if (warp == 0) {
      if (lane == 0 && all > 0) {
        bool ok = true;
        mbar_arrive_expect_tx(&sh.q_full, 2 * T::kQ);
        for (int q = 0; q < 2; ++q)
          for (int b = 0; b < kBlocks; ++b)
            load_tile(smem + q * T::kQ + b * 16384, &maps.q, maps.q_swap, 64 * b, head, q0 + first + q * kTileQ,
                      &sh.q_full);
        // Unit 2 j is key tile j, unit 2 j + 1 value tile j.  `used` blocks have been
        // given out since the start, `freed` given back.
        int unit = 0, gone = 0, used = 0, freed = 0, at = 0;
        for (; unit < 2 * all && ok; ++unit) {
          const int j = unit >> 1, n = unit & 1 ? vb : kBlocks;
          while (ok && used + n - freed > T::kRing) {
            ok = mbar_wait(&sh.empty[gone % kUnits], (gone / kUnits) & 1);
            freed += gone & 1 ? vb : kBlocks;
            ++gone;
          }
          if (!ok) break;
          uint64_t* full = &sh.full[unit % kUnits];
          mbar_arrive_expect_tx(full, n * T::kBlock);
          for (int b = 0; b < n; ++b) {
            uint8_t* dst = ring + at * T::kBlock;
            if (unit & 1) load_tile(dst, &maps.v, maps.v_swap, 128 * part + 64 * b, head, k0 + j * kKeys, full);
            else if (b < kBlocks - 1) load_tile(dst, &maps.k, maps.k_swap, 64 * b, head, k0 + j * kKeys, full);
            else tma_load_2d(dst, &maps.r, 0, k0 + j * kKeys, full);
            if (++at == T::kRing) at = 0;
          }
          used += n;
        }
        // Copies still in flight land before the CTA's memory is given back.
        mbar_wait(&sh.q_full, 0);
        for (int u = max(0, unit - kUnits); u < unit; ++u) mbar_wait(&sh.full[u % kUnits], (u / kUnits) & 1);
      }
    } else if (warp == 1) {
      const uint32_t score_desc = half_idesc(kAct == kBF16, kKeys, a.scale < 0.0f, false, false);
      const uint32_t value_desc = half_idesc(kAct == kBF16, 64 * vb, false, false, true);
      const uint32_t half_desc = half_idesc(kAct == kBF16, 64, false, false, true);
      const uint32_t td = uniform(tmem), sq = uniform(desc_lo_sw128(smem_u32(smem))),
                     sk = uniform(desc_lo_sw128(smem_u32(ring))),
                     sv = uniform(desc_lo_rows128(smem_u32(ring), T::kBlock));
      const int n0 = uniform(tiles[0]), n1 = uniform(tiles[1]), steps = max(n0, n1);
      bool ok = steps == 0 || warp_wait(&sh.q_full, 0);
      int at = 0;  // the block after the last tile's
      // The blocks of the next tile, as low words of their descriptors.
      auto blocks = [&](uint32_t base, int n, uint32_t* lo) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (b >= n) break;
          lo[b] = uniform(base + at * (T::kBlock >> 4));
          if (++at == T::kRing) at = 0;
        }
      };
      // S_q of a key tile.
      auto scores = [&](int q, const uint32_t* kt) {
        const uint32_t qt = sq + q * (T::kQ >> 4);
        if (elect_one()) {
#pragma unroll
          for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc_mma_f16(td + q * 128, desc_of(qt + ((b * 16384 + kk * 32) >> 4)), desc_of(kt[b] + (kk * 32 >> 4)),
                         score_desc, (b | kk) != 0);
          tc_commit(&sh.s_full[q]);
        }
        __syncwarp();
      };
      uint32_t kt[4], vt[4];
      if (ok && steps > 0) ok = warp_wait(&sh.full[0], 0);
      if (ok && steps > 0) {
        tc_fence_after();
        blocks(sk, kBlocks, kt);
        if (n0 > 0) scores(0, kt);
        if (n1 > 0) scores(1, kt);
        if (elect_one()) tc_commit(&sh.empty[0]);
        __syncwarp();
      }
      for (int j = 0; j < steps && ok; ++j) {
        const int unit = 2 * j + 1;
        ok = warp_wait(&sh.full[unit % kUnits], (unit / kUnits) & 1);
        if (!ok) break;
        const int first_block = at;
        blocks(sv, vb, vt);
        const int valid = uniform(keys) - j * kKeys;
        if (valid < kKeys) {  // rows behind the sequence's last key
          for (int b = 0; b < vb; ++b) {
            uint8_t* tile = ring + (first_block + b < T::kRing ? first_block + b : first_block + b - T::kRing) * T::kBlock;
            for (int i = lane; i < (kKeys - valid) * 8; i += 32)
              reinterpret_cast<uint4*>(tile + valid * 128)[i] = make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
          __syncwarp();
        }
        const bool joined = vb == 1 || first_block + 1 < T::kRing;  // the value blocks lie in a row
        const bool more = j + 1 < steps;
        bool next = !more;  // key tile j + 1 has arrived
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int n = q ? n1 : n0;
          if (!ok || j >= n) continue;
          ok = warp_wait(&sh.p_ready[q], j & 1);
          if (!ok) continue;
          tc_fence_after();
          if (elect_one()) {
            if (joined) {
#pragma unroll
              for (int kk = 0; kk < kKeys / 16; ++kk)
                tc_mma_f16_ts(td + 256 + q * 128, td + q * 128 + kk * 8, desc_of(vt[0] + (kk * 2048 >> 4)), value_desc,
                              kk > 0 || j > 0);
            } else {
#pragma unroll
              for (int kk = 0; kk < kKeys / 16; ++kk)
#pragma unroll
                for (int b = 0; b < 2; ++b)
                  tc_mma_f16_ts(td + 256 + q * 128 + 64 * b, td + q * 128 + kk * 8, desc_of(vt[b] + (kk * 2048 >> 4)),
                                half_desc, kk > 0 || j > 0);
            }
            if (j + 1 >= n) tc_commit(&sh.o_done[q]);
            if (q == 1 || j >= n1) tc_commit(&sh.empty[unit % kUnits]);  // the value tile's last use
          }
          __syncwarp();
          if (!next) {
            ok = warp_wait(&sh.full[(unit + 1) % kUnits], ((unit + 1) / kUnits) & 1);
            tc_fence_after();
            blocks(sk, kBlocks, kt);
            next = true;
          }
          if (ok && j + 1 < n) scores(q, kt);
        }
        if (ok && more && elect_one()) tc_commit(&sh.empty[(unit + 1) % kUnits]);
        __syncwarp();
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
    const int q = (warp - 4) / 4, quad = warp & 3;
    const int row = first + q * kTileQ + quad * 32 + lane;
    const int seen = row < queries ? min(keys - queries + 1 + row, keys) : 0;
    const uint32_t lanes = static_cast<uint32_t>(32 * quad) << 16;
    const uint32_t ts = tmem + lanes + q * 128, to = tmem + lanes + 256 + q * 128;
    const float c = fmaxf(fabsf(a.scale), 1e-30f) * 1.4426950408889634f;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int j = 0; j < tiles[q]; ++j) {
      ok = mbar_wait(&sh.s_full[q], j & 1);
      if (!ok) break;
      tc_fence_after();
      uint32_t s[kKeys];
#pragma unroll
      for (int i = 0; i < kKeys; i += 32) tc_ld32(ts + i, s + i);
      tc_wait_ld();
      tc_settle<kKeys>(s);
      const int left = seen - j * kKeys;
      if (__any_sync(0xffffffffu, left < kKeys)) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
          if (i >= left) s[i] = 0xff800000u;
      }
      // The largest score of the row so far.
      auto largest = [&]() {
        float top[4] = {m, m, m, m};
#pragma unroll
        for (int i = 0; i < kKeys; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(s[i]));
        return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      };
      // The weights of the tile against the present m, into tensor memory over
      // the scores; their sum, and the largest exponent (before the lift).
      float sum, grown;
      auto weigh = [&]() {
        const float base = m == -INFINITY ? 0.0f : kLift - m * c;
        const uint64_t scale2 = both(c, c), base2 = both(base, base);
        uint64_t part[2] = {0, 0};
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kKeys; i += 32) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint64_t xy =
                fma2(both(__uint_as_float(s[i + 2 * e]), __uint_as_float(s[i + 2 * e + 1])), scale2, base2);
            float x, y, u, v;
            apart(xy, x, y);
            top[e & 1] = fmaxf(top[e & 1], fmaxf(x, y));
            u = exp2_fast(x);
            v = exp2_fast(y);
            part[e & 1] = add2(part[e & 1], both(u, v));
            p[e] = pack<kAct>(u, v);
          }
          tc_st16(ts + i / 2, p);
        }
        float s0, s1, s2, s3;
        apart(part[0], s0, s1);
        apart(part[1], s2, s3);
        sum = (s0 + s1) + (s2 + s3);
        grown = fmaxf(top[0], top[1]);
      };
      if (j == 0) m = largest();
      weigh();
      // Rarely a score has outgrown m: raise it, multiply what was summed, weigh
      // the tile again.  PV of tile j - 1 is complete (this tile's scores were
      // committed after it).
      if (j > 0 && __any_sync(0xffffffffu, grown > kLift + kLag || (m == -INFINITY && grown > -INFINITY))) {
        const float best = largest();
        const float keep = best > m ? exp2_fast((m - best) * c) : 1.0f;
        m = best;
        l *= keep;
#pragma unroll 1
        for (int i = 0; i < 64 * vb; i += 32) {
          uint32_t o[32];
          tc_ld32(to + i, o);
          tc_wait_ld();
          tc_settle<32>(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
          tc_st32(to + i, o);
        }
        weigh();
      }
      l += sum;
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&sh.p_ready[q]);
    }
    if (tiles[q] > 0 && ok) ok = mbar_wait(&sh.o_done[q], 0);
    tc_fence_after();
    const bool store = row < queries;
    const int64_t at = (static_cast<int64_t>(q0) + row) * a.heads + head;
    if (a.lse && part == 0 && store)
      a.lse[at] = !ok ? NAN : l > 0.0f ? (m * c - kLift + log2f(l)) * 0.6931471805599453f : (l == 0.0f ? -INFINITY : l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    for (int i = 0; i < 64 * vb; i += 32) {
      uint32_t o[32];
      if (tiles[q] > 0) {
        tc_ld32(to + i, o);
        tc_wait_ld();
        tc_settle<32>(o);
      }
      if (!store) continue;
      uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at * a.value + 128 * part + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t w[4];
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          float u = __uint_as_float(o[8 * e + 2 * f]) * inv, v = __uint_as_float(o[8 * e + 2 * f + 1]) * inv;
          if (seen <= 0) u = v = 0.0f;
          if (!ok) u = v = __int_as_float(0x7fc00000);
          w[f] = pack<kAct>(u, v);
        }
        dst[e] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_free(tmem, 512);
}

// A map over [tokens][heads][channels] rows, boxes of 64 channels x `rows`
// tokens; the two outer dimensions in ascending order of their strides.
bool encode_rows(CUtensorMap* map, int* swap, CUtensorMapDataType type, const void* base, int channels, int heads,
                 int64_t tokens, int64_t token_stride, int64_t head_stride, uint32_t rows) {
  const uint64_t least = (static_cast<uint64_t>(channels) * 2 + 15) / 16 * 16;
  uint64_t hs = heads > 1 ? static_cast<uint64_t>(head_stride) * 2 : least;
  uint64_t ts = tokens > 1 ? static_cast<uint64_t>(token_stride) * 2 : hs * heads;
  *swap = ts < hs;
  const uint64_t n = static_cast<uint64_t>(tokens), h = static_cast<uint64_t>(heads), d = static_cast<uint64_t>(channels);
  if (*swap) return encode_tiled_3d(map, type, base, {d, n, h}, {ts, hs}, {64, rows, 1}, CU_TENSOR_MAP_SWIZZLE_128B);
  return encode_tiled_3d(map, type, base, {d, h, n}, {hs, ts}, {64, 1, rows}, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int kAct, int kBlocks>
cudaError_t launch(const LatentPromptArgs& a, cudaStream_t s) {
  using T = Tiles<kBlocks>;
  const CUtensorMapDataType type =
      kAct == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  Maps maps;
  // Without keys no tile is loaded; the maps then describe the queries.
  const bool empty = a.total_k == 0;
  const int64_t keys = empty ? a.total_q : a.total_k;
  if (!encode_rows(&maps.q, &maps.q_swap, type, a.q, a.nope + kLatentRope, a.heads, a.total_q, a.q_token, a.q_head,
                   kTileQ) ||
      !encode_rows(&maps.k, &maps.k_swap, type, empty ? a.q : a.k, empty ? 64 : a.nope, a.heads, keys,
                   empty ? a.q_token : a.k_token, empty ? a.q_head : a.k_head, T::kKeys) ||
      !encode_tiled_2d(&maps.r, type, empty ? a.q : a.k_rope, 64, keys,
                       2 * (empty ? a.q_token : (keys > 1 ? a.kr_token : 64)), 64, T::kKeys,
                       CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_rows(&maps.v, &maps.v_swap, type, empty ? a.q : a.v, empty ? 64 : a.value, a.heads, keys,
                   empty ? a.q_token : a.v_token, empty ? a.q_head : a.v_head, T::kKeys))
    return cudaErrorInvalidValue;
  auto kernel = latent_prompt_kernel<kAct, kBlocks>;
  static std::atomic<uint64_t> ready{0};
  cudaError_t err = allow_shared_memory(kernel, kSmem + 1024, ready);
  if (err != cudaSuccess) return err;
  const int parts = (a.value + 127) / 128;
  const int64_t tiles = (a.total_q + 255) / 256 + a.seqs;
  return launch_pdl(kernel, dim3(static_cast<unsigned>(tiles * a.heads * parts)), dim3(kThreads), kSmem + 1024, s, maps,
                    a, parts);
}

template <int kAct>
cudaError_t launch_blocks(const LatentPromptArgs& a, cudaStream_t s) {
  if (a.nope == 64) return launch<kAct, 2>(a, s);
  if (a.nope == 128) return launch<kAct, 3>(a, s);
  return launch<kAct, 4>(a, s);
}

}  // namespace

cudaError_t launch_latent_prompt(const LatentPromptArgs& a, cudaStream_t s) {
  if (a.total_q == 0) return cudaSuccess;
  return a.dtype == kF16 ? launch_blocks<kF16>(a, s) : launch_blocks<kBF16>(a, s);
}

}  // namespace exlr8
