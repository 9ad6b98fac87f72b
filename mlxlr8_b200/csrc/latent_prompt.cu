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
// without a pass for its maximum first, and P stays below 2^14 and float16
// weights keep their full precision down to 2^-20 of the largest.  P is rounded to
// the operands' type for the second product, which takes no wider one beside
// 16-bit values (the output's error grows by 22 to 30%); l is of the unrounded.
//
// Tensor memory is full: S_0, S_1, O_0, O_1 of 128 columns each, P_q over S_q.
// While the threads of one query tile form its weights the tensor pipe works for
// the other one, which is why two tiles share a CTA (and why each K and V tile
// is read from L2 once for 256 queries).
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
// four give up.  Value channels beyond 128 are a second CTA's (the scores are
// formed again there).  Rows of the last key tile that belong to no key of the
// sequence are zeroed in the V tile, since 0 x NaN would reach the sum.  Waits
// are bounded; one that runs out leaves NaN in the CTA's output.
//
// Where the tiles of queries are few, a cluster of two to eight CTAs shares the
// keys of one: each leaves O, m and l of its share in its shared memory, float32
// over the operands, and joins a part of the rows from all of them, in the order
// of the shares.
//
// A tile of at most 128 queries leaves one query tile empty: its key tiles go to
// the two softmax groups in turn, so that the products of one run under the
// weights of the other (82 queries of six sequences over 2000 keys each, 24
// heads: 40 -> 28 us).
//
// 8192 queries of 32 heads (128 + 64 key and 128 value channels): 549 us in a
// burst at 1965 MHz, 1252 TFLOP/s, and 634 us, 1084 TFLOP/s, at the 1520 MHz that
// the power cap leaves after a second, the tensor pipe bound; 5 prompts of 1300
// tokens, 16 heads: 25 us, the longest one's keys in turn (2900 cycles a tile for
// 256 queries).

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
  // Of eight units in a row three at least are key tiles, the others a block each.
  static_assert(3 * kBlocks + 5 > kRing, "kUnits units lie in the ring at once");
};

constexpr int kSplitGroups = 80;  // tiles of queries from which no two CTAs per tile would fit the GPU

constexpr int kUnits = 8;  // key and value tiles that the barriers tell apart

struct Shared {
  uint64_t q_full, full[kUnits], empty[kUnits];
  uint64_t s_full[2], p_ready[2], o_done[2];
  uint32_t tmem;
  int tile, q0, queries, k0, keys;  // tile -1: none
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

// Four floats at the same shared-memory place of CTA `rank` of the cluster.
__device__ __forceinline__ float4 load_cluster4(const void* p, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr(smem_u32(p), rank)));
  return v;
}
__device__ __forceinline__ float2 load_cluster2(const void* p, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(cluster_addr(smem_u32(p), rank)));
  return v;
}

__device__ __forceinline__ float4 join(const float4& a, float f, const float4& b, float g) {
  return make_float4(fmaf(a.x, f, b.x * g), fmaf(a.y, f, b.y * g), fmaf(a.z, f, b.z * g), fmaf(a.w, f, b.w * g));
}

// Lane and lane ^ off exchange: the one without the bit keeps its x and takes the
// other's x for y, the one with it keeps its y and takes the other's y for x.
__device__ __forceinline__ void trade(uint4& x, uint4& y, bool bit, int off) {
  uint32_t* const u = &x.x;
  uint32_t* const v = &y.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, bit ? u[i] : v[i], off);
    if (bit) u[i] = other;
    else v[i] = other;
  }
}

// kSplit: a cluster shares the keys of one tile of queries.
template <int kAct, int kBlocks, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
    latent_prompt_kernel(const __grid_constant__ Maps maps, const LatentPromptArgs a, int value_parts, int shares) {
  using T = Tiles<kBlocks>;
  constexpr int kKeys = T::kKeys;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared sh;
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* const ring = smem + 2 * T::kQ;
  float4* const staged = reinterpret_cast<float4*>(smem);  // [256][128 channels] of a share, over the operands
  float2* const stats = reinterpret_cast<float2*>(smem + 256 * 512);        // of its rows: unit of O (log2), sum
  float* const weights = reinterpret_cast<float*>(smem + 256 * 512 + 2048);  // [128][8] of the rows that it joins
  const int warp = static_cast<int>(uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const int columns = a.heads * value_parts;
  const int group = kSplit ? blockIdx.x / shares : blockIdx.x, share = kSplit ? blockIdx.x % shares : 0;
  const int head = group % columns / value_parts, part = group % value_parts;

  // The CTA's sequence and its tile of 256 queries: tiles are numbered over
  // the sequences and taken from the last (its rows see the most keys).
  pdl_launch_dependents();
  pdl_wait();
  if (warp == 0) {
    // A sequence's queries and keys, one sequence a lane.
    int q0, queries, k0, keys;
    auto load = [&](int s) {
      auto clamped = [](int v, int64_t total) { return min(max(v, 0), static_cast<int>(total)); };
      const bool some = s < a.seqs;
      q0 = some ? clamped(a.q_starts[s], a.total_q) : 0;
      k0 = some ? clamped(a.k_starts[s], a.total_k) : 0;
      queries = some ? max(clamped(a.q_starts[s + 1], a.total_q) - q0, 0) : 0;
      keys = some ? max(clamped(a.k_starts[s + 1], a.total_k) - k0, 0) : 0;
    };
    int total = 0;
    for (int s0 = 0; s0 < a.seqs; s0 += 32) {
      load(s0 + lane);
      total += __reduce_add_sync(0xffffffffu, (queries + 255) / 256);
    }
    int at = total - 1 - group / columns, tile = -1;
    for (int s0 = 0; s0 < a.seqs && at >= 0 && tile < 0; s0 += 32) {
      if (a.seqs > 32) load(s0 + lane);
      const int n = (queries + 255) / 256;
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
        q0 = __shfl_sync(0xffffffffu, q0, which);
        k0 = __shfl_sync(0xffffffffu, k0, which);
        queries = __shfl_sync(0xffffffffu, queries, which);
        keys = __shfl_sync(0xffffffffu, keys, which);
      } else {
        at -= __shfl_sync(0xffffffffu, end, 31);
      }
    }
    if (lane == 0) {
      sh.tile = tile;
      sh.q0 = q0, sh.queries = queries, sh.k0 = k0, sh.keys = keys;
      prefetch_tensor_map(&maps.q);
      prefetch_tensor_map(&maps.k);
      prefetch_tensor_map(&maps.r);
      prefetch_tensor_map(&maps.v);
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
  if (warp == 1) tmem_alloc(&sh.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  if (sh.tile < 0) {
    if (warp == 1) tmem_free(tmem, 512);
    return;
  }
  const int q0 = sh.q0, queries = sh.queries, k0 = sh.k0, keys = sh.keys;
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
  int begin = 0;  // the first key tile of this CTA's share
  if (kSplit) {
    const int most = max(tiles[0], tiles[1]);
    begin = most * share / shares;
    const int end = most * (share + 1) / shares;
#pragma unroll
    for (int q = 0; q < 2; ++q) tiles[q] = max(min(tiles[q], end) - begin, 0);
  }
  const int all = max(tiles[0], tiles[1]);
  // One query tile alone: both softmax groups take its key tiles in turn, each
  // with a maximum, a sum and an output of its own, joined at the end.
  const bool lone = first + kTileQ >= queries;
  const int own0 = k0 + begin * kKeys;  // the share's first key
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
    if (warp == 0) {
      if (lane == 0 && all > 0) {
        bool ok = true;
        mbar_arrive_expect_tx(&sh.q_full, lone ? T::kQ : 2 * T::kQ);
        for (int q = 0; q < (lone ? 1 : 2); ++q)
          for (int b = 0; b < kBlocks; ++b)
            load_tile(smem + q * T::kQ + b * 16384, &maps.q, maps.q_swap, 64 * b, head, q0 + first + q * kTileQ,
                      &sh.q_full);
        // Units in the order of their use: K_0 V_0 K_1 V_1 ..., for a lone query tile
        // K_0 K_1 V_0 K_2 V_1 ... V_n-2 V_n-1.  `used` blocks have been given out
        // since the start, `freed` given back.
        const int units = 2 * all;
        auto is_value = [&](int u) { return !lone ? (u & 1) != 0 : u + 1 == units || (u > 0 && (u & 1) == 0); };
        int unit = 0, gone = 0, used = 0, freed = 0, at = 0;
        for (; unit < units && ok; ++unit) {
          const bool value = is_value(unit);
          const int n = value ? vb : kBlocks;
          const int j = !lone ? unit / 2 : value ? (unit + 1 == units ? all : unit / 2) - 1 : (unit + 1) / 2;
          while (ok && used + n - freed > T::kRing) {
            ok = mbar_wait(&sh.empty[gone % kUnits], (gone / kUnits) & 1);
            freed += is_value(gone) ? vb : kBlocks;
            ++gone;
          }
          if (!ok) break;
          uint64_t* full = &sh.full[unit % kUnits];
          mbar_arrive_expect_tx(full, n * T::kBlock);
          for (int b = 0; b < n; ++b) {
            uint8_t* dst = ring + at * T::kBlock;
            if (value) load_tile(dst, &maps.v, maps.v_swap, 128 * part + 64 * b, head, own0 + j * kKeys, full);
            else if (b < kBlocks - 1) load_tile(dst, &maps.k, maps.k_swap, 64 * b, head, own0 + j * kKeys, full);
            else tma_load_2d(dst, &maps.r, 0, own0 + j * kKeys, full);
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
        const uint32_t qt = sq + (lone ? 0 : q) * (T::kQ >> 4);
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
      // The blocks of value tile j; rows behind the sequence's last key are zeroed.
      // Whether they lie in a row.
      auto values = [&](int j) {
        const int first_block = at;
        blocks(sv, vb, vt);
        const int valid = uniform(keys - begin * kKeys) - j * kKeys;
        if (valid < kKeys) {
          for (int b = 0; b < vb; ++b) {
            const int block = first_block + b < T::kRing ? first_block + b : first_block + b - T::kRing;
            for (int i = lane; i < (kKeys - valid) * 8; i += 32)
              reinterpret_cast<uint4*>(ring + block * T::kBlock + valid * 128)[i] = make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
          __syncwarp();
        }
        return vb == 1 || first_block + 1 < T::kRing;
      };
      // O_q (+)= P_q V; one thread.
      auto product = [&](int q, bool joined, bool more) {
        if (joined) {
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            tc_mma_f16_ts(td + 256 + q * 128, td + q * 128 + kk * 8, desc_of(vt[0] + (kk * 2048 >> 4)), value_desc,
                          kk > 0 || more);
        } else {
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
#pragma unroll
            for (int b = 0; b < 2; ++b)
              tc_mma_f16_ts(td + 256 + q * 128 + 64 * b, td + q * 128 + kk * 8, desc_of(vt[b] + (kk * 2048 >> 4)),
                            half_desc, kk > 0 || more);
        }
      };
      if (lone) {
        int unit = 1;
        // The next unit, a key tile, against Q_0 into S_q.
        auto next_scores = [&](int q) {
          ok = warp_wait(&sh.full[unit % kUnits], (unit / kUnits) & 1);
          if (!ok) return;
          tc_fence_after();
          blocks(sk, kBlocks, kt);
          scores(q, kt);
          if (elect_one()) tc_commit(&sh.empty[unit % kUnits]);
          __syncwarp();
          ++unit;
        };
        if (ok && steps > 1) next_scores(1);
        for (int j = 0; j < steps && ok; ++j) {
          const int q = j & 1;
          ok = warp_wait(&sh.full[unit % kUnits], (unit / kUnits) & 1);
          if (!ok) break;
          const bool joined = values(j);
          ok = warp_wait(&sh.p_ready[q], (j >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            product(q, joined, j > 1);
            if (j + 2 >= steps) tc_commit(&sh.o_done[q]);
            tc_commit(&sh.empty[unit % kUnits]);
          }
          __syncwarp();
          ++unit;
          if (j + 2 < steps) next_scores(q);
        }
      } else {
        for (int j = 0; j < steps && ok; ++j) {
          const int unit = 2 * j + 1;
          ok = warp_wait(&sh.full[unit % kUnits], (unit / kUnits) & 1);
          if (!ok) break;
          const bool joined = values(j);
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
              product(q, joined, j > 0);
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
    }
    if constexpr (kSplit) {
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
    const int q = (warp - 4) / 4, quad = warp & 3;
    const int row = first + (lone ? 0 : q) * kTileQ + quad * 32 + lane;
    const int count = !lone ? tiles[q] : (all + 1 - q) / 2;  // key tiles of this group
    const int seen = (row < queries ? min(keys - queries + 1 + row, keys) : 0) - begin * kKeys;  // of the share
    const uint32_t lanes = static_cast<uint32_t>(32 * quad) << 16;
    const uint32_t ts = tmem + lanes + q * 128, to = tmem + lanes + 256 + q * 128;
    const float c = fmaxf(fabsf(a.scale), 1e-30f) * 1.4426950408889634f;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int t = 0; t < count; ++t) {
      const int j = lone ? 2 * t + q : t;
      ok = warp_wait(&sh.s_full[q], t & 1);
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
      if (t == 0) m = largest();
      weigh();
      // Rarely a score has outgrown m: raise it, multiply what was summed, weigh
      // the tile again.  PV of the group's last tile is complete (this tile's scores
      // were committed after it).
      if (t > 0 && __any_sync(0xffffffffu, grown > kLift + kLag || (m == -INFINITY && grown > -INFINITY))) {
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
    if (count > 0 && ok) ok = warp_wait(&sh.o_done[q], 0);
    tc_fence_after();
    // A lone tile's second group, and every CTA of a cluster, leaves its output in
    // shared memory, over the operand tiles once both groups are done with them;
    // 16-byte pieces swizzled by the row.
    float unit = m * c - kLift, other = 0.0f, own = 1.0f;  // what O counts, log2; the parts' factors
    const int r = q * kTileQ + quad * 32 + lane;
    auto stage = [&](bool add) {
      for (int i = 0; i < 64 * vb; i += 32) {
        uint32_t o[32];
        tc_ld32(to + i, o);
        tc_wait_ld();
        tc_settle<32>(o);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float4 v = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]),
                                 __uint_as_float(o[4 * e + 3]));
          if (add) v = join(v, own, staged[(r + kTileQ) * 32 + ((i / 4 + e) ^ (r & 7))], other);
          staged[r * 32 + ((i / 4 + e) ^ (r & 7))] = v;
        }
      }
    };
    const bool both = lone && all > 1;  // the same for all threads
    if (kSplit || both) asm volatile("bar.sync 1, 256;" ::: "memory");
    if (both) {
      if (q == 1) {
        stats[r] = make_float2(unit, ok ? l : NAN);
        stage(false);
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (q == 0) {
        const float2 v = stats[r + kTileQ];
        const float top = fmaxf(l != 0.0f ? unit : -INFINITY, v.y != 0.0f ? v.x : -INFINITY);
        own = l != 0.0f ? exp2_fast(unit - top) : 0.0f;
        other = v.y != 0.0f ? exp2_fast(v.x - top) : 0.0f;
        l = l * own + v.y * other;
        unit = top;
      }
    }
    if constexpr (kSplit) {
      // (rows of a lone tile's second group are no query's)
      if (!(lone && q == 1)) {
        stats[r] = make_float2(unit, ok ? l : NAN);
        if (count > 0) stage(both);
      }
      __syncwarp();
      cluster_sync();
      // A CTA joins its share of the rows: first what each CTA's part of a row
      // counts (eight lanes a row), then the parts, a warp a row.
      const int row0 = 256 * share / shares, rows = 256 * (share + 1) / shares - row0;
      const int id = threadIdx.x - 128;
      for (int i0 = 0; i0 < rows; i0 += 32) {
        const int i = i0 + id / 8, s = id % 8;
        const bool there = i < rows && s < shares;
        const float2 v = there ? load_cluster2(&stats[row0 + i], s) : make_float2(0.0f, 0.0f);
        float top = v.y != 0.0f ? v.x : -INFINITY;
#pragma unroll
        for (int off = 4; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float f = v.y != 0.0f ? exp2_fast(v.x - top) : 0.0f;
        float sum = v.y * f;
#pragma unroll
        for (int off = 4; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (i < rows) weights[i * 8 + s] = v.y != 0.0f ? f / sum : 0.0f;
        const int at = first + row0 + i;
        if (a.lse && part == 0 && i < rows && s == 0 && at < queries)
          a.lse[(static_cast<int64_t>(q0) + at) * a.heads + head] =
              sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
      }
      __syncwarp();
      asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll 2
      for (int i = warp - 4; i < rows; i += 8) {
        const int r = row0 + i, at = first + r;
        if (at >= queries || lane >= 16 * vb) continue;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int s0 = 0; s0 < shares; s0 += 4) {
          float4 p[4];
#pragma unroll
          for (int s = 0; s < 4; ++s)
            p[s] = load_cluster4(&staged[r * 32 + (lane ^ (r & 7))], min(s0 + s, shares - 1));
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const float f = weights[i * 8 + s0 + s];
            if (f == 0.0f) continue;  // a part that sees nothing of the row holds no output
            sum.x = fmaf(p[s].x, f, sum.x);
            sum.y = fmaf(p[s].y, f, sum.y);
            sum.z = fmaf(p[s].z, f, sum.z);
            sum.w = fmaf(p[s].w, f, sum.w);
          }
        }
        reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) +
                                 ((static_cast<int64_t>(q0) + at) * a.heads + head) * a.value + 128 * part)[lane] =
            make_uint2(pack<kAct>(sum.x, sum.y), pack<kAct>(sum.z, sum.w));
      }
      __syncwarp();
      cluster_sync();  // no CTA leaves while its part is read
    } else if (!(lone && q == 1)) {
      const bool store = row < queries;
      const int64_t at = (static_cast<int64_t>(q0) + row) * a.heads + head;
      if (a.lse && part == 0 && store)
        a.lse[at] = !ok ? NAN : l > 0.0f ? (unit + log2f(l)) * 0.6931471805599453f : (l == 0.0f ? -INFINITY : l);
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      for (int i = 0; i < 64 * vb; i += 32) {
        uint32_t o[32];
        if (count > 0) {
          tc_ld32(to + i, o);
          tc_wait_ld();
          tc_settle<32>(o);
        }
        if (both) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 p = staged[(r + kTileQ) * 32 + ((i / 4 + e) ^ (r & 7))];
            o[4 * e] = __float_as_uint(fmaf(__uint_as_float(o[4 * e]), own, p.x * other));
            o[4 * e + 1] = __float_as_uint(fmaf(__uint_as_float(o[4 * e + 1]), own, p.y * other));
            o[4 * e + 2] = __float_as_uint(fmaf(__uint_as_float(o[4 * e + 2]), own, p.z * other));
            o[4 * e + 3] = __float_as_uint(fmaf(__uint_as_float(o[4 * e + 3]), own, p.w * other));
          }
        }
        uint4 w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t two[4];
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            float u = __uint_as_float(o[8 * e + 2 * f]) * inv, v = __uint_as_float(o[8 * e + 2 * f + 1]) * inv;
            if (seen <= 0) u = v = 0.0f;
            if (!ok) u = v = __int_as_float(0x7fc00000);
            two[f] = pack<kAct>(u, v);
          }
          w[e] = make_uint4(two[0], two[1], two[2], two[3]);
        }
        // Four lanes trade pieces of their rows, so that they store 64 bytes of
        // one row at a time (a row a lane took 3500 cycles for 256 x 128).
        trade(w[0], w[1], lane & 1, 1);
        trade(w[2], w[3], lane & 1, 1);
        trade(w[0], w[2], lane & 2, 2);
        trade(w[1], w[3], lane & 2, 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t to_row = row - (lane & 3) + e;
          if (to_row < queries)
            reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + ((q0 + to_row) * a.heads + head) * a.value +
                                     128 * part + i)[lane & 3] = w[e];
        }
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

// Clusters of n CTAs that the current device holds at once; asked of the driver
// once per device and size.
template <typename Kernel>
cudaError_t clusters_at_once(Kernel kernel, cudaLaunchConfig_t cfg, int n, int* clusters) {
  static std::atomic<int> known[16][9];
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  if (device < 16 && (*clusters = known[device][n].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
  cfg.gridDim = dim3(n);
  cfg.attrs->val.clusterDim.x = n;
  err = cudaOccupancyMaxActiveClusters(clusters, kernel, &cfg);
  if (err == cudaSuccess && device < 16) known[device][n].store(*clusters, std::memory_order_relaxed);
  return err;
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
  const int parts = (a.value + 127) / 128;
  // No more tiles of 256 queries can hold queries of ascending sequences.
  const int64_t tiles = a.total_q < a.seqs ? a.total_q : (a.total_q - a.seqs) / 256 + a.seqs;
  const int64_t groups = tiles * a.heads * parts;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(groups));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem + 1024;
  cfg.stream = s;
  static std::atomic<uint64_t> ready[2];
  // Few tiles of queries leave SMs idle while each walks its keys one tile after
  // the other: a cluster of CTAs shares them, as many as are resident at once,
  // two key tiles each at least (165 queries over 2165 keys, 8 heads of 256 + 256
  // channels: 58 us alone, 29 by four, 24 by six; by eight, of which 15 fit and 16
  // were needed, 35).
  int shares = 1;
  const int64_t key_tiles = a.total_k / a.seqs / T::kKeys;
  if (groups < kSplitGroups && key_tiles >= 4) {
    auto kernel = latent_prompt_kernel<kAct, kBlocks, true>;
    cudaError_t err = allow_shared_memory(kernel, kSmem + 1024, ready[1]);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    for (int n = 8, fit; err == cudaSuccess && n > 1 && shares == 1; --n) {
      if (2 * n > key_tiles) continue;
      err = clusters_at_once(kernel, cfg, n, &fit);
      if (groups <= fit) shares = n;
    }
    if (err != cudaSuccess) return err;
    if (shares > 1) {
      attr[0].val.clusterDim.x = shares;
      cfg.gridDim.x = static_cast<unsigned>(groups * shares);
      cfg.numAttrs = 2;
      return cudaLaunchKernelEx(&cfg, kernel, maps, a, parts, shares);
    }
  }
  auto kernel = latent_prompt_kernel<kAct, kBlocks, false>;
  const cudaError_t err = allow_shared_memory(kernel, kSmem + 1024, ready[0]);
  if (err != cudaSuccess) return err;
  cfg.attrs = attr + 1;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, maps, a, parts, 1);
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
