// Attention over the paged latent cache (absorbed form): every head of a
// query attends the same row [c_j, k_j] of a token,
//   s_j = scale * (ql . c_j + qr . k_j),  out = sum_j softmax(s)_j c_j.
// Query t of T sees the first length - T + 1 + t tokens; a query that sees
// none gives zeros (and lse -inf).  Table entries outside the cache hold no
// tokens.
//
// The rows (query, head) of a sequence are the narrow side, so both products
// are taken transposed, with 64 tokens or 128 latent channels on the tensor
// core's M side and kN = 16, 32 or 64 rows on its N side:
//   S^T [64 tokens][kN]   = C Q^T       cache tile as loaded (channels contiguous)
//   P^T = 2^(c S^T + base)              one thread per token, float32, to shared memory
//   O^T [rank][kN]       += C^T P^T     the same tile, taken with its tokens contracted
// A cache tile is read from memory once and feeds both products.  base = 6 -
// c m with c = |scale| log2(e) (a negative scale negates the cache tile in the
// instruction) and m a row's maximum when it was last raised: it is raised,
// and O and the sums multiplied, only when a score has grown past it by 2^8,
// so a tile needs no maximum over its tokens, only the vote that none has.
// Weights stay below 2^14 and float16 ones keep full precision down to 2^-20
// of the largest.  They are rounded to the operands' type for the second product,
// which takes no wider ones beside 16-bit values (the output's error grows by 6
// to 18%); their sums are float32, of the unrounded weights.
//
// Work is the flat list of (sequence, row tile, 64 tokens), cut evenly over
// the CTAs (one per SM) whatever the lengths; a sequence cut in two or more
// leaves float32 parts in the workspace, which a second kernel joins, in the
// order of the list.
//
// Warp 0 loads (TMA; one box per page or 16 to 64 of its tokens), warps 1 and 2
// issue the two products, so that the scores of the next tile are formed while
// this one's weights are; warps 4-7 and 8-11 each take half of the rows for the
// 64 tokens.  Tiles of 64 tokens, not 128, because the queries (72 KB at 64
// rows of 576) leave room for 2 tiles of 64 but not for two of 128: with one
// tile of 128 nothing overlapped and a tile's chain of load, scores, weights
// and product was the bound (167 us for 64 sequences of up to 12000 tokens).  The
// latent is loaded as pairs of 64-channel blocks (one M = 128 of the second
// product) into a ring; a pair is given back as soon as its product is done.
// The second product takes the steps of 16 tokens that hold one; token rows
// among them that belong to no token are zeroed in the tile, since 0 x NaN would
// reach the sum.  Waits are bounded; one that runs out leaves NaN in the rows
// that it concerns.
//
// 64 heads of rank 512, bfloat16: 64 sequences of up to 12000 tokens 137 us (4.9
// TB/s of cache; HBM bound but for the first and last tiles and the join, 7 us) in
// a burst at 1965 MHz, 158 us at the 1600 MHz that the power cap leaves after a
// second; one of 16000 18.5 us (parts written and joined, 10 us of it).

#include <cuda.h>

#include "common.cuh"
#include "latent.cuh"
#include "launch.cuh"
#include "tensor_map.cuh"
#include "umma.cuh"

namespace exlr8 {

namespace {

constexpr int kThreads = 384;
constexpr int kTile = 64;  // tokens
constexpr float kLift = 6.0f;
constexpr float kLag = 8.0f;
constexpr uint32_t kBlock = kTile * 128;  // 64 tokens x 64 channels
constexpr uint32_t kPair = 2 * kBlock;
constexpr int kMaxStages = 4;       // tiles in the ring
constexpr int kMaxPairs = 4 * kMaxStages;
constexpr uint32_t kSmem = 232448;  // all of a CTA's shared memory

// ---- the flat list of tiles -----------------------------------------------------

struct Work {
  int64_t batch;
  int queries, heads, row_tiles;
  int64_t room;  // tokens a table holds
  const int32_t* lengths;
};

__device__ __forceinline__ int tokens_of(const Work& w, int64_t b) {
  return static_cast<int>(min(static_cast<int64_t>(max(w.lengths[b], 0)), w.room));
}
__device__ __forceinline__ int tiles_of(const Work& w, int64_t b) { return (tokens_of(w, b) + kTile - 1) / kTile; }

// The list that the CTAs share: every (sequence, row tile) has its tiles and
// `extra` further places that stand for what a segment costs besides them
// (queries, first scores, output), where shares are long enough to be evened
// out (21 sequences of up to 291 tokens and 320 rows: 30 us without, 26 with; 3 of
// up to 28084 and 40 rows: 36 and 34; 64 of up to 12000 and 64 rows: 138 both).
struct List {
  int64_t total, sharers;  // places, CTAs
  int extra;
};
constexpr int kSegmentCost = 2;

// The calling warp takes part as a whole.  A CTA takes two tiles at least, where
// one each would cut sequences in more than half as many places as there are
// CTAs (the parts are what a short call spends its time on: 9 sequences of up to
// 1167 tokens and 64 rows, 25 us with two and 29 with one; 5 of up to 700 and 60
// rows, 23 and 19).
__device__ List list_of(const Work& w, int ctas, int lane) {
  int64_t n = 0, sequences = 0;
  for (int64_t b = lane; b < w.batch; b += 32) {
    const int tiles = tiles_of(w, b);
    n += tiles;
    sequences += tiles > 0;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    n += __shfl_xor_sync(0xffffffffu, n, off);
    sequences += __shfl_xor_sync(0xffffffffu, sequences, off);
  }
  n *= w.row_tiles;
  sequences *= w.row_tiles;
  const int64_t least = n - sequences > ctas / 2 ? 2 : 1, most = (n + least - 1) / least;
  const int extra = n > 2 * ctas ? kSegmentCost : 0;
  return List{n + extra * sequences, most < ctas ? most : ctas, extra};
}

// A place of the list: its sequence and row tile, that one's first place, the
// tile (its number of tiles: one of the extra places), and the tiles before it.
struct Spot {
  int64_t sequence, start, before;
  int rt, tile, tokens, tiles;
};
__device__ Spot find_place(const Work& w, const List& list, int64_t at, int lane) {
  int64_t base = 0, sequences = 0;
  for (int64_t b0 = 0; b0 < w.batch; b0 += 32) {
    const int64_t b = b0 + lane;
    const int tokens = b < w.batch ? tokens_of(w, b) : 0, tiles = (tokens + kTile - 1) / kTile;
    const int64_t n = tiles > 0 ? static_cast<int64_t>(tiles + list.extra) * w.row_tiles : 0;
    int64_t end = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t other = __shfl_up_sync(0xffffffffu, end, off);
      if (lane >= off) end += other;
    }
    const uint32_t some = __ballot_sync(0xffffffffu, tiles > 0), mine = __ballot_sync(0xffffffffu, at < base + end);
    if (mine) {
      const int which = __ffs(mine) - 1;
      Spot p;
      p.sequence = b0 + which;
      p.tokens = __shfl_sync(0xffffffffu, tokens, which);
      p.tiles = __shfl_sync(0xffffffffu, tiles, which);
      p.start = base + __shfl_sync(0xffffffffu, end - n, which);
      sequences += __popc(some & ((1u << which) - 1));
      p.before = p.start - list.extra * w.row_tiles * sequences;
      p.tile = static_cast<int>(at - p.start);
      p.rt = 0;
      if (w.row_tiles > 1) {
        const int64_t unit = p.tiles + list.extra;
        p.rt = static_cast<int>((at - p.start) / unit);
        p.tile = static_cast<int>((at - p.start) % unit);
        p.start += p.rt * unit;
        p.before += static_cast<int64_t>(p.rt) * p.tiles;
      }
      p.tile = min(p.tile, p.tiles);
      p.before += p.tile;
      return p;
    }
    base += __shfl_sync(0xffffffffu, end, 31);
    sequences += __popc(some);
  }
  return Spot{w.batch, base, base - list.extra * w.row_tiles * sequences, 0, 0, 0, 0};
}

// The first place of CTA i of n that share `total`.
__device__ __forceinline__ int64_t first_tile(int64_t i, int64_t total, int64_t n) {
  // (a 64-bit division takes longer than the lists that need one are common)
  if (total < (1 << 20)) return static_cast<uint32_t>(i) * static_cast<uint32_t>(total) / static_cast<uint32_t>(n);
  return i * total / n;
}

// The CTA of place x: the last whose first place is not behind it.
__device__ __forceinline__ int64_t owner_of(int64_t x, int64_t total, int64_t n) {
  if (total < (1 << 20)) return (static_cast<uint32_t>(x + 1) * static_cast<uint32_t>(n) - 1) / static_cast<uint32_t>(total);
  return ((x + 1) * n - 1) / total;
}

// A CTA's walk over its share: one segment per (sequence, row tile).
struct Walk {
  int64_t b, left;    // sequence, tiles of the share not yet taken
  int rt, tile;       // row tile, first tile of the next segment
  int tokens, tiles;  // of the sequence
  int begin, end;     // the segment's tiles
  __device__ __forceinline__ bool next(const Work& w) {
    if (left <= 0) return false;
    while (tile >= tiles) {  // on to the next row tile, then the next sequence that has tokens
      tile = 0;
      if (tiles == 0 || ++rt >= w.row_tiles) {
        rt = 0;
        if (++b >= w.batch) return false;
        tokens = tokens_of(w, b);
        tiles = (tokens + kTile - 1) / kTile;
      }
    }
    begin = tile;
    end = static_cast<int>(min(static_cast<int64_t>(tiles), begin + left));
    left -= end - begin;
    tile = end;
    return true;
  }
};

// What a CTA that begins inside a (sequence, row tile) leaves for the join: the
// CTAs that share it, `first` to first + count - 1, and the slot of the part of
// the first; count is 0 where the CTA begins with one.
struct Cut {
  int64_t sequence;
  int rt, first, count, slot;
};

// ---- the main kernel -------------------------------------------------------------

struct Layout {
  uint32_t q, p, rope, ring, shared;  // byte offsets in shared memory; P is two deep
  int stages, ropes;                  // whole tiles in the ring; rotary buffers, 1 or 2
};

struct Shared {
  uint64_t q_full, q_empty, o_done, s_full[2], s_empty[2], p_ready[2], p_done[2];
  uint64_t full[kMaxPairs], empty[kMaxPairs], rope_full[2], rope_empty[2];
  uint32_t tmem;
  Walk walk;
  List list;
  int64_t start;  // first place of the (sequence, row tile) in which the share begins
  __align__(16) float base[64];
  __align__(16) float factor[64];
  float m[64];
  float top[4][64];
  int limit[64];
};

static_assert(sizeof(Shared) <= 3072, "leaves room for two tiles of rank 512 beside 64 rows");

// A tile of the ring and the parity of its round.  (Counted, not divided, and
// of whole tiles, so that the issuing warps add constants to one base a tile:
// with a division, and later a broadcast, per pair they were the bound.)
struct Place {
  int stage = 0;
  uint32_t round = 0;
  __device__ __forceinline__ void advance(int stages) {
    if (++stage == stages) {
      stage = 0;
      round ^= 1;
    }
  }
};

struct Maps {
  CUtensorMap q, r, cache;
};

// (by whole warps, like the barrier of a vote below)
__device__ __forceinline__ void group_sync(int id) {
  __syncwarp();
  asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory");
}
__device__ __forceinline__ bool group_any(int id, bool v) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n bar.red.or.pred q, %1, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"(id), "r"(static_cast<uint32_t>(v))
      : "memory");
  return r != 0;
}

// A sum of weighted rows over the sum of its weights: 0 for a query that saw no
// token, also where 0 times a row that is not finite made the sum NaN.
__device__ __forceinline__ float share(uint32_t sum, float factor) {
  return factor == 0.0f ? 0.0f : __uint_as_float(sum) * factor;
}

template <int kCols>
__device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t (&v)[kCols]) {
  if constexpr (kCols == 32) tc_ld32(taddr, v);
  else if constexpr (kCols == 16) tc_ld16(taddr, v);
  else tc_ld8(taddr, v);
}
template <int kCols>
__device__ __forceinline__ void store_columns(uint32_t taddr, const uint32_t (&v)[kCols]) {
  if constexpr (kCols == 32) tc_st32(taddr, v);
  else if constexpr (kCols == 16) tc_st16(taddr, v);
  else tc_st8(taddr, v);
}

// Value `own` of the 16 lanes of a half warp folded together, own = lane % 16 /
// (16 / kN): every step halves the values a lane holds.
template <int kN, class F>
__device__ __forceinline__ float fold(const float (&v)[kN], int lane, F f) {
  float t[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) t[i] = v[i];
#pragma unroll
  for (int m = kN / 2, off = 8; off > 0; m /= 2, off /= 2) {
    const bool up = lane & off;
    if (m == 0) t[0] = f(t[0], __shfl_xor_sync(0xffffffffu, t[0], off));
#pragma unroll
    for (int i = 0; i < m; ++i) {
      const float other = __shfl_xor_sync(0xffffffffu, up ? t[i] : t[i + m], off);
      t[i] = f(up ? t[i + m] : t[i], other);
    }
  }
  return t[0];
}

// A CTA leaves two parts at most: slot i holds that of CTA i's first segment,
// slot CTAs + i that of its last.  parts: [2 * CTAs][kN][rank] float32, sums:
// [kN][2 * CTAs] pairs (log2 of the unit of O and the sum, the sum).
template <int kAct, int kN>
__global__ void __launch_bounds__(kThreads, 1)
    latent_attention_kernel(const __grid_constant__ Maps maps, const LatentAttentionArgs a, const Work w,
                            const Layout lay, int box, uint32_t columns, float* __restrict__ parts, float2* __restrict__ sums,
                            Cut* __restrict__ cuts) {
  pdl_launch_dependents();
  extern __shared__ __align__(1024) uint8_t smem[];  // (nothing static lies before it)
  Shared& sh = *reinterpret_cast<Shared*>(smem + lay.shared);
  const int warp = static_cast<int>(uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const int blocks = a.rank / 64, tile_pairs = a.rank / 128;
  if (warp == 0) {
    pdl_wait();
    const List list = list_of(w, gridDim.x, lane);
    Walk walk{};
    if (blockIdx.x < list.sharers) {
      const int64_t next = first_tile(blockIdx.x + 1, list.total, list.sharers);
      const Spot p = find_place(w, list, first_tile(blockIdx.x, list.total, list.sharers), lane);
      const int64_t end = list.extra > 0 ? find_place(w, list, next, lane).before : next;
      walk = Walk{p.sequence, end - p.before, p.rt, p.tile, p.tokens, p.tiles, 0, 0};
      if (lane == 0) {
        sh.list = list;
        sh.start = p.start;
      }
    }
    if (lane == 0) sh.walk = walk;
  } else if (warp == 1) {
    tmem_alloc(&sh.tmem, columns);
  } else if (warp == 2 && lane == 0) {
    prefetch_tensor_map(&maps.q);
    prefetch_tensor_map(&maps.r);
    prefetch_tensor_map(&maps.cache);
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_empty, 1);
    mbar_init(&sh.o_done, 1);
    for (int i = 0; i < kMaxPairs; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.rope_full[i], 1);
      mbar_init(&sh.rope_empty[i], 1);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.s_empty[i], 256);
      mbar_init(&sh.p_ready[i], 256);
      mbar_init(&sh.p_done[i], 1);
    }
    mbar_fence_init();
  } else if (warp > 2) {
    // Sequences without tokens are no CTA's work: their rows are zeroed here.
    pdl_wait();
    const int64_t rows = static_cast<int64_t>(a.queries) * a.heads;
    for (int64_t b = blockIdx.x; b < a.batch; b += gridDim.x) {
      if (tokens_of(w, b) > 0) continue;
      for (int64_t i = threadIdx.x - 96; i < rows * a.rank / 8; i += kThreads - 96)
        reinterpret_cast<uint4*>(a.out)[b * (rows * a.rank / 8) + i] = make_uint4(0, 0, 0, 0);
      if (a.lse)
        for (int64_t i = threadIdx.x - 96; i < rows; i += kThreads - 96) a.lse[b * rows + i] = -INFINITY;
    }
  }
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  Walk walk = sh.walk;
  const uint32_t tmem = sh.tmem, t_scores = tmem + tile_pairs * kN;
  bool ok = true;

  if (warp == 0) {
    int u = 0, segment = 0, loaded = 0;  // tiles, segments and pairs so far
    Place place;
    for (; ok && walk.next(w); ++segment) {
      if (segment > 0) ok = warp_wait(&sh.q_empty, (segment - 1) & 1);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&sh.q_full, (blocks + 1) * kN * 128);
        for (int i = 0; i < blocks; ++i)
          tma_load_3d(smem + lay.q + i * kN * 128, &maps.q, 64 * i, walk.rt * kN, static_cast<int>(walk.b), &sh.q_full);
        tma_load_3d(smem + lay.q + blocks * kN * 128, &maps.r, 0, walk.rt * kN, static_cast<int>(walk.b), &sh.q_full);
      }
      for (int t = walk.begin; ok && t < walk.end; ++t, ++u) {
        // Lane i fetches the tokens [i * box, (i + 1) * box) of the tile.
        const int token = t * kTile + lane * box;
        int row = -1;
        if (lane * box < kTile && token < walk.tokens) {
          const int page = a.block_table[walk.b * a.table_width + token / a.page_size];
          if (page >= 0 && page < a.pages) row = page * a.page_size + token % a.page_size;
        }
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, row >= 0)) * box * 128;
        for (int i = 0; ok && i < tile_pairs; ++i, ++loaded) {
          const int slot = place.stage * tile_pairs + i;
          uint64_t* full = &sh.full[slot];
          ok = warp_wait(&sh.empty[slot], place.round ^ 1);  // (passes in the first round)
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(full, 2 * bytes);
          __syncwarp();
          if (row >= 0) {
            uint8_t* dst = smem + lay.ring + slot * kPair + lane * box * 128;
            tma_load_2d(dst, &maps.cache, 128 * i, row, full);
            tma_load_2d(dst + kBlock, &maps.cache, 128 * i + 64, row, full);
          }
        }
        if (!ok) break;
        place.advance(lay.stages);
        const int r = u & (lay.ropes - 1);
        ok = warp_wait(&sh.rope_empty[r], ((u >> (lay.ropes - 1)) & 1) ^ 1);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&sh.rope_full[r], bytes);
        __syncwarp();
        if (row >= 0) tma_load_2d(smem + lay.rope + r * kBlock + lane * box * 128, &maps.cache, a.rank, row, &sh.rope_full[r]);
      }
    }
    // Copies still in flight land before the CTA's memory is given back.
    if (segment > 0) mbar_wait(&sh.q_full, (segment - 1) & 1);
    const int slots = lay.stages * tile_pairs;
    for (int i = max(0, loaded - slots); i < loaded; ++i) mbar_wait(&sh.full[i % slots], (i / slots) & 1);
    for (int i = max(0, u - lay.ropes); i < u; ++i)
      mbar_wait(&sh.rope_full[i & (lay.ropes - 1)], (i >> (lay.ropes - 1)) & 1);
  } else if (warp == 1) {  // scores
    const uint32_t desc = half_idesc(kAct == kBF16, kN, a.scale < 0.0f, false, false, kTile);
    const uint32_t ts = uniform(t_scores), sq = uniform(desc_lo_sw128(smem_u32(smem + lay.q))),
                   sc = uniform(desc_lo_sw128(smem_u32(smem + lay.ring))),
                   sr = uniform(desc_lo_sw128(smem_u32(smem + lay.rope)));
    int u = 0;
    Place place;
    for (int segment = 0; ok && uniform(walk.next(w)); ++segment) {
      const int begin = uniform(walk.begin), end = uniform(walk.end);
      ok = warp_wait(&sh.q_full, segment & 1);
      for (int t = begin; ok && t < end; ++t, ++u) {
        const int r = u & 1;
        const uint32_t to = uniform(ts + r * kN);
        ok = warp_wait(&sh.s_empty[r], ((u >> 1) & 1) ^ 1);  // (passes in the first round)
        const uint32_t ct = uniform(sc + place.stage * (tile_pairs * (kPair >> 4)));
#pragma unroll
        for (int i = 0; i < kLatentMaxRank / 128; ++i) {
          if (i >= tile_pairs || !ok) continue;
          ok = warp_wait(&sh.full[place.stage * tile_pairs + i], place.round);
          if (!ok) continue;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              tc_mma_f16(to, desc_of(ct + ((i * kPair + (k / 4) * kBlock + (k % 4) * 32) >> 4)),
                         desc_of(sq + (((2 * i + k / 4) * kN * 128 + (k % 4) * 32) >> 4)), desc, k > 0 || i > 0);
          }
          __syncwarp();
        }
        place.advance(lay.stages);
        const int rope = u & (lay.ropes - 1);
        if (ok) ok = warp_wait(&sh.rope_full[rope], (u >> (lay.ropes - 1)) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t rt = uniform(sr + rope * (kBlock >> 4)), qr = sq + blocks * (kN * 128 >> 4);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_f16(to, desc_of(rt + (k * 32 >> 4)), desc_of(qr + (k * 32 >> 4)), desc, 1);
          tc_commit(&sh.s_full[r]);
          tc_commit(&sh.rope_empty[rope]);
          if (t + 1 == end) tc_commit(&sh.q_empty);
        }
        __syncwarp();
      }
    }
  } else if (warp == 2) {  // products with the weights
    const uint32_t desc = half_idesc(kAct == kBF16, kN, false, true, true);
    const uint32_t td = uniform(tmem), sp = uniform(desc_lo_rows128(smem_u32(smem + lay.p), kBlock)),
                   sv = uniform(desc_lo_rows128(smem_u32(smem + lay.ring), kBlock));
    int u = 0;
    Place place;
    while (ok && uniform(walk.next(w))) {
      const int begin = uniform(walk.begin), end = uniform(walk.end);
      for (int t = begin; ok && t < end; ++t, ++u) {
        ok = warp_wait(&sh.p_ready[u & 1], (u >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t pt = uniform(sp + (u & 1) * (kBlock >> 4));
        const uint32_t ct = uniform(sv + place.stage * (tile_pairs * (kPair >> 4)));
        const int steps = uniform((walk.tokens - t * kTile + 15) / 16);  // 16 tokens each
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < kLatentMaxRank / 128; ++i) {
            if (i >= tile_pairs) continue;
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k)
              if (k < steps)
                tc_mma_f16(td + i * kN, desc_of(ct + ((i * kPair + k * 2048) >> 4)), desc_of(pt + (k * 2048 >> 4)),
                           desc, k > 0 || t > begin);
            tc_commit(&sh.empty[place.stage * tile_pairs + i]);
          }
          tc_commit(&sh.p_done[u & 1]);
          if (t + 1 == end) tc_commit(&sh.o_done);
        }
        __syncwarp();
        place.advance(lay.stages);
      }
    }
  } else if (warp == 3) {  // what the join needs to know
    if (lane == 0) {
      Cut cut{walk.b, walk.rt, 0, 0, 0};
      if (walk.tile > 0 && walk.tile < walk.tiles) {
        const List list = sh.list;
        cut.first = static_cast<int>(owner_of(sh.start, list.total, list.sharers));
        cut.count =
            static_cast<int>(owner_of(sh.start + walk.tiles - 1, list.total, list.sharers)) - cut.first + 1;
        // (tiles of its own before these, not only extra places)
        const bool second = first_tile(cut.first, list.total, list.sharers) < sh.start - list.extra;
        cut.slot = cut.first + (second ? gridDim.x : 0);
      }
      cuts[blockIdx.x] = cut;
    }
  } else if (warp >= 4) {
    constexpr int kCols = kN / 2;
    // Tensor memory has a quarter's 16 tokens in lanes 0 to 15; lanes 16 to 31
    // take half of their rows over, so that lane i has token i % 16 and kOwn rows.
    constexpr int kOwn = kCols / 2, kShare = 16 / kOwn;
    const int half = (warp - 4) / 4, quad = warp & 3, bar = 1 + half;
    const int token_row = quad * 16 + (lane & 15), col0 = half * kCols, own0 = col0 + (lane >> 4) * kOwn;
    const uint32_t lanes = static_cast<uint32_t>(32 * quad) << 16;
    const float c = fmaxf(fabsf(a.scale), 1e-30f) * 1.4426950408889634f;
    const int rows = a.queries * a.heads;
    int u = 0;
    Place place;
    for (int segment = 0; walk.next(w); ++segment) {
      // One warp of each half keeps its rows' maxima and limits.
      if (quad == 0 && lane < kCols) {
        const int row = walk.rt * kN + col0 + lane;
        sh.base[col0 + lane] = INFINITY;
        sh.m[col0 + lane] = -INFINITY;
        sh.limit[col0 + lane] = row < rows ? walk.tokens - a.queries + 1 + row / a.heads : walk.tokens;
      }
      group_sync(bar);
      const int least = walk.tokens - a.queries + 1 + walk.rt * kN / a.heads;
      float l[kOwn];
#pragma unroll
      for (int i = 0; i < kOwn; ++i) l[i] = 0.0f;
      for (int t = walk.begin; t < walk.end; ++t, ++u, place.advance(lay.stages)) {
        const int token = t * kTile + token_row, r = u & 1;
        bool held = token < walk.tokens;
        if (held) {
          const int page = a.block_table[walk.b * a.table_width + token / a.page_size];
          held = page >= 0 && page < a.pages;
        }
        if (ok) ok = mbar_wait(&sh.s_full[r], (u >> 1) & 1);
        tc_fence_after();
        uint32_t all[kCols];
        load_columns<kCols>(t_scores + lanes + r * kN + col0, all);
        tc_wait_ld();
        tc_settle<kCols>(all);
        tc_fence_before();
        mbar_arrive(&sh.s_empty[r]);
        float s[kOwn];
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          const uint32_t other = __shfl_sync(0xffffffffu, all[kOwn + i], lane & 15);
          s[i] = __uint_as_float(lane < 16 ? all[i] : other);
        }
        // P's buffer is free once the products of the tile before the last are done.
        if (ok && u > 1) ok = mbar_wait(&sh.p_done[r], ((u >> 1) - 1) & 1);
        if (!held && ok && token < (walk.tokens + 15) / 16 * 16) {
          // The two lanes of a token zero half of this half's blocks each, in an
          // order that spreads a warp's tokens over the banks.
          uint8_t* tile = smem + lay.ring + place.stage * tile_pairs * kPair + token_row * 128;
          for (int i = half * blocks / 2; i < (half + 1) * blocks / 2; ++i) {
            uint4* line = reinterpret_cast<uint4*>(tile + i * kBlock);
#pragma unroll
            for (int e = 0; e < 4; ++e) line[((lane >> 4) * 4 + e) ^ (token_row & 7)] = make_uint4(0, 0, 0, 0);
          }
        }
        if (__any_sync(0xffffffffu, !held || token >= least)) {
#pragma unroll
          for (int i = 0; i < kOwn; ++i)
            if (!held || token >= sh.limit[own0 + i]) s[i] = -INFINITY;
        }
        float base[kOwn];
        float grown = -INFINITY;
#pragma unroll
        for (int i = 0; i < kOwn; i += 4) {
          const float4 v = *reinterpret_cast<const float4*>(&sh.base[own0 + i]);
          base[i] = v.x, base[i + 1] = v.y, base[i + 2] = v.z, base[i + 3] = v.w;
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i) grown = fmaxf(grown, fmaf(s[i], c, base[i]));
        if (group_any(bar, grown > kLift + kLag)) {
          const float best = fold(s, lane, [](float a, float b) { return fmaxf(a, b); });
          if (lane % kShare == 0) sh.top[quad][own0 + lane % 16 / kShare] = best;
          group_sync(bar);
          if (quad == 0 && lane < kCols) {
            const int i = col0 + lane;
            const float old = sh.m[i];
            const float m = fmaxf(fmaxf(fmaxf(sh.top[0][i], sh.top[1][i]), fmaxf(sh.top[2][i], sh.top[3][i])), old);
            sh.m[i] = m;
            sh.factor[i] = m > old ? exp2_fast((old - m) * c) : 1.0f;
            sh.base[i] = m == -INFINITY ? INFINITY : kLift - m * c;
          }
          group_sync(bar);
#pragma unroll
          for (int i = 0; i < kOwn; ++i) {
            l[i] *= sh.factor[own0 + i];
            base[i] = sh.base[own0 + i];
          }
          if (t > walk.begin) {
            if (ok) ok = mbar_wait(&sh.p_done[r ^ 1], ((u - 1) >> 1) & 1);  // the products of the tile before
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < tile_pairs; ++k) {
              uint32_t o[kCols];
              load_columns<kCols>(tmem + lanes + k * kN + col0, o);
              tc_wait_ld();
              tc_settle<kCols>(o);
#pragma unroll
              for (int i = 0; i < kCols; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * sh.factor[col0 + i]);
              store_columns<kCols>(tmem + lanes + k * kN + col0, o);
            }
            tc_wait_st();
          }
        }
        uint32_t p[kOwn / 2];
#pragma unroll
        for (int i = 0; i < kOwn; i += 2) {
          // a row without a maximum has only hidden tokens: -inf + inf would be NaN
          const float p0 = exp2_fast(fmaf(s[i], c, base[i] == INFINITY ? 0.0f : base[i]));
          const float p1 = exp2_fast(fmaf(s[i + 1], c, base[i + 1] == INFINITY ? 0.0f : base[i + 1]));
          l[i] += p0;
          l[i + 1] += p1;
          p[i / 2] = pack<kAct>(p0, p1);
        }
        // Row `token` of P, 16-byte pieces swizzled by the token.
        uint8_t* line = smem + lay.p + r * kBlock + token_row * 128;
        if constexpr (kOwn >= 8) {
#pragma unroll
          for (int i = 0; i < kOwn; i += 8)
            *reinterpret_cast<uint4*>(line + ((((own0 + i) / 8) ^ (token_row & 7)) * 16)) =
                make_uint4(p[i / 2], p[i / 2 + 1], p[i / 2 + 2], p[i / 2 + 3]);
        } else {
          *reinterpret_cast<uint2*>(line + (((own0 / 8) ^ (token_row & 7)) * 16) + (own0 & 4) * 2) = make_uint2(p[0], p[1]);
        }
        fence_async_smem();
        tc_fence_before();
        mbar_arrive(&sh.p_ready[r]);
      }
      // The segment's sums over the tokens, then its output.
      const float row_sum = fold(l, lane, [](float a, float b) { return a + b; });
      if (lane % kShare == 0) sh.top[quad][own0 + lane % 16 / kShare] = row_sum;
      group_sync(bar);
      const bool whole = walk.begin == 0 && walk.end == walk.tiles;
      const int64_t slot = blockIdx.x + (segment > 0 ? gridDim.x : 0);
      if (quad == 0 && lane < kCols) {
        const int i = col0 + lane, row = walk.rt * kN + i;
        const float sum = (sh.top[0][i] + sh.top[1][i]) + (sh.top[2][i] + sh.top[3][i]);
        const float unit = sh.m[i] * c - kLift;
        if (!whole) sums[i * 2 * gridDim.x + slot] = make_float2(unit, ok ? sum : NAN);
        else if (a.lse && row < rows)
          a.lse[walk.b * rows + row] = !ok ? NAN : sum == 0.0f ? -INFINITY : (unit + log2f(sum)) * 0.6931471805599453f;
        sh.factor[i] = !ok ? NAN : sum == 0.0f ? 0.0f : 1.0f / sum;
      }
      group_sync(bar);
      if (ok) ok = mbar_wait(&sh.o_done, segment & 1);
      tc_fence_after();
      for (int k = 0; k < tile_pairs; ++k) {
        uint32_t o[kCols];
        load_columns<kCols>(tmem + lanes + k * kN + col0, o);
        tc_wait_ld();
        tc_settle<kCols>(o);
        if (!ok) {
#pragma unroll
          for (int i = 0; i < kCols; ++i) o[i] = 0x7fc00000u;
        }
        const int channel = 128 * k + quad * 32 + lane;
        if (!whole) {
          float* dst = parts + (slot * kN + col0) * a.rank + channel;
          const int count = rows - walk.rt * kN - col0;  // (the join reads no row past the last)
#pragma unroll
          for (int i = 0; i < kCols; ++i, dst += a.rank)
            if (i < count) *dst = __uint_as_float(o[i]);
        } else {
          // Four lanes trade their channels of four rows, so that each stores four
          // channels of one (single channels took 8000 cycles at 64 x 512).
          const int row = walk.rt * kN + col0 + (lane & 3);
          uint2* dst = reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (walk.b * rows + row) * a.rank +
                                                (channel & ~3));
#pragma unroll
          for (int i = 0; i < kCols; i += 4, dst += a.rank) {
            const float4 f = *reinterpret_cast<const float4*>(&sh.factor[col0 + i]);
            const uint32_t two[2] = {pack<kAct>(share(o[i], f.x), share(o[i + 1], f.y)),
                                     pack<kAct>(share(o[i + 2], f.z), share(o[i + 3], f.w))};
            uint32_t w[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {  // channels c, c + 1 of row 2 e + lane % 2
              const uint32_t other = __shfl_xor_sync(0xffffffffu, two[e], 1);
              w[e] = lane & 1 ? __byte_perm(other, two[e], 0x7632) : __byte_perm(two[e], other, 0x5410);
            }
            const uint32_t other = __shfl_xor_sync(0xffffffffu, lane & 2 ? w[0] : w[1], 2);
            if (row + i < rows) *dst = lane & 2 ? make_uint2(other, w[1]) : make_uint2(w[0], other);
          }
        }
      }
      group_sync(bar);  // the shared rows are free for the next segment
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_free(tmem, columns);
}

// ---- joining the parts ---------------------------------------------------------------

constexpr int kJoinWarps = 8;
constexpr int kJoinShare = 4;   // CTAs per cut
constexpr int kJoinHeld = 5;    // parts of a row a lane weighs
constexpr int kMaxCtas = 32 * kJoinHeld;

// A sequence is cut where a CTA's share begins inside it, and its cuts divide
// its rows among themselves: blockIdx.y + 1 is that CTA, blockIdx.x one of the
// four that divide them again.  A warp takes a row, 16 channels a lane; with
// more CTAs than rows, a CTA takes 128 channels of a row and its warps share
// the parts.  (A row's cuts are neighbours in the grid, so that those with work
// are resident at once.)
template <int kAct>
__global__ void __launch_bounds__(32 * kJoinWarps, 4)
    latent_join_kernel(const LatentAttentionArgs a, const Work w, int kn, const float* __restrict__ parts,
                       const float2* __restrict__ sums, const Cut* __restrict__ cuts) {
  __shared__ float4 s_o[kJoinWarps][32];
  __shared__ float s_f[kJoinWarps][32 * kJoinHeld];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t cta = blockIdx.y + 1;
  const Cut cut = cuts[cta];
  if (cut.count == 0) return;
  // A part lies in its CTA's first slot where the share begins with the
  // sequence or inside it, in the second where it ends with its beginning.
  const int ctas = gridDim.y + 1, first = cut.first, count = cut.count;
  auto slot_of = [&](int k) { return k == 0 ? cut.slot : first + k; };
  const int rows = w.queries * w.heads, vectors = a.rank / 128;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int workers = (count - 1) * kJoinShare;
  const int worker = (static_cast<int>(cta) - first - 1) * kJoinShare + blockIdx.x;
  // The largest unit of a row's parts, their sum, and what each part counts
  // (in s_f[warp]); the whole warp.
  auto weigh = [&](int i, float& top, float& sum) {
    float2 v[kJoinHeld];
    top = -INFINITY;
    sum = 0.0f;
#pragma unroll
    for (int e = 0; e < kJoinHeld; ++e) {
      const int k = lane + 32 * e;
      v[e] = k < count ? sums[i * 2 * ctas + slot_of(k)] : make_float2(0.0f, 0.0f);
    }
#pragma unroll
    for (int e = 0; e < kJoinHeld; ++e)
      if (v[e].y != 0.0f) top = fmaxf(top, v[e].x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    __syncwarp();
#pragma unroll
    for (int e = 0; e < kJoinHeld; ++e) {
      const float f = v[e].y != 0.0f ? exp2_fast(v[e].x - top) : 0.0f;
      sum = fmaf(v[e].y, f, sum);
      s_f[warp][lane + 32 * e] = f;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    __syncwarp();
  };
  auto add = [](float4& o, const float4& p, float f) {
    o.x = fmaf(p.x, f, o.x);
    o.y = fmaf(p.y, f, o.y);
    o.z = fmaf(p.z, f, o.z);
    o.w = fmaf(p.w, f, o.w);
  };
  auto store = [&](int row, int vector, const float4& o, float inv) {
    uint2* dst = reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (cut.sequence * rows + row) * a.rank);
    dst[32 * vector + lane] = inv == 0.0f ? make_uint2(0, 0)  // (see share)
                                          : make_uint2(pack<kAct>(o.x * inv, o.y * inv), pack<kAct>(o.z * inv, o.w * inv));
  };
  float top, sum;
  if (kn > workers) {
    for (int i = worker + warp * workers; i < kn; i += kJoinWarps * workers) {
      const int row = cut.rt * kn + i;
      if (row >= rows) break;
      weigh(i, top, sum);
      float4 o[kLatentMaxRank / 128] = {};
#pragma unroll 4
      for (int k = 0; k < count; ++k) {
        const int at = slot_of(k) * kn + i;
        const float f = s_f[warp][k];
        const float4* part = reinterpret_cast<const float4*>(parts + static_cast<int64_t>(at) * a.rank) + lane;
#pragma unroll
        for (int e = 0; e < kLatentMaxRank / 128; ++e)
          if (e < vectors) add(o[e], part[32 * e], f);
      }
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      if (a.lse && lane == 0)
        a.lse[cut.sequence * rows + row] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
#pragma unroll
      for (int e = 0; e < kLatentMaxRank / 128; ++e)
        if (e < vectors) store(row, e, o[e], inv);
    }
    return;
  }
  for (int unit = worker; unit < kn * vectors; unit += workers) {
    const int i = unit / vectors, vector = unit % vectors, row = cut.rt * kn + i;
    if (row >= rows) break;
    weigh(i, top, sum);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int k = warp; k < count; k += kJoinWarps) {
      const int at = slot_of(k) * kn + i;
      add(o, *(reinterpret_cast<const float4*>(parts + static_cast<int64_t>(at) * a.rank) + 32 * vector + lane),
          s_f[warp][k]);
    }
    s_o[warp][lane] = o;
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int g = 1; g < kJoinWarps; ++g) add(o, s_o[g][lane], 1.0f);
      store(row, vector, o, sum == 0.0f ? 0.0f : 1.0f / sum);
      if (a.lse && lane == 0 && vector == 0)
        a.lse[cut.sequence * rows + row] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
    }
    __syncthreads();
  }
}

int rows_per_tile(int rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms < kMaxCtas ? sms : kMaxCtas;
}

// Two tiles in the ring let the next one land and be scored while this one is
// weighed; with 1.75 (two rotary buffers at 64 rows of rank 512) every tile
// waited for its last pair (64 sequences of up to 12000 tokens: 202 us, not 178).
Layout layout(int rank, int kn) {
  Layout l{};
  l.q = 0;
  l.p = (rank / 64 + 1) * kn * 128;  // a multiple of 1 KB: kn * 128 is one of 2 KB
  l.rope = l.p + 2 * kBlock;
  for (l.ropes = 2;; --l.ropes) {
    l.ring = l.rope + l.ropes * kBlock;
    l.stages = static_cast<int>((kSmem - sizeof(Shared) - l.ring) / (rank / 128 * kPair));
    if (l.stages >= 2 || l.ropes == 1) break;
  }
  if (l.stages > kMaxStages) l.stages = kMaxStages;
  l.shared = l.ring + l.stages * (rank / 128) * kPair;
  return l;
}

template <int kAct, int kN>
cudaError_t launch(const LatentAttentionArgs& a, cudaStream_t s) {
  const CUtensorMapDataType type =
      kAct == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const int rows = a.queries * a.heads, row_tiles = (rows + kN - 1) / kN, ctas = sm_count();
  const Work w{a.batch, a.queries, a.heads, row_tiles,
               a.pages > 0 ? static_cast<int64_t>(a.table_width) * a.page_size : 0, a.lengths};
  float* parts = static_cast<float*>(a.workspace);
  float2* sums = reinterpret_cast<float2*>(parts + 2ll * ctas * kN * a.rank);
  Cut* cuts = reinterpret_cast<Cut*>(sums + 2ll * ctas * kN);
  // The largest power of two (16 to 64) that divides a page: no box crosses one.
  int box = 16;
  while (box < kTile && a.page_size % (2 * box) == 0) box *= 2;
  Maps maps;
  const uint64_t n = static_cast<uint64_t>(rows), b = static_cast<uint64_t>(a.batch), d = static_cast<uint64_t>(a.rank);
  // Without pages nothing is loaded; the map then describes the queries.
  const bool empty = w.room == 0;
  if (!encode_tiled_3d(&maps.q, type, a.q_latent, {d, n, b}, {d * 2, d * n * 2}, {64, kN, 1},
                       CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_tiled_3d(&maps.r, type, a.q_rope, {64, n, b}, {128, 128 * n}, {64, kN, 1}, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_tiled_2d(&maps.cache, type, empty ? a.q_latent : a.cache, empty ? d : d + kLatentRope,
                       empty ? n : static_cast<uint64_t>(a.pages) * a.page_size, 2 * (empty ? d : d + kLatentRope), 64,
                       box, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  uint32_t columns = 32;
  while (columns < static_cast<uint32_t>(kN * (a.rank / 128 + 2))) columns *= 2;
  auto kernel = latent_attention_kernel<kAct, kN>;
  static std::atomic<uint64_t> ready{0};
  cudaError_t err = allow_shared_memory(kernel, kSmem, ready);
  if (err != cudaSuccess) return err;
  const Layout lay = layout(a.rank, kN);
  err = launch_pdl(kernel, dim3(ctas), dim3(kThreads), lay.shared + sizeof(Shared), s, maps, a, w, lay, box, columns,
                   parts, sums, cuts);
  if (err != cudaSuccess || ctas < 2) return err;
  return launch_pdl(latent_join_kernel<kAct>, dim3(kJoinShare, ctas - 1), dim3(32 * kJoinWarps), 0, s, a, w, kN,
                    static_cast<const float*>(parts), static_cast<const float2*>(sums),
                    static_cast<const Cut*>(cuts));
}

template <int kAct>
cudaError_t launch_rows(const LatentAttentionArgs& a, cudaStream_t s) {
  switch (rows_per_tile(a.queries * a.heads)) {
    case 16: return launch<kAct, 16>(a, s);
    case 32: return launch<kAct, 32>(a, s);
    default: return launch<kAct, 64>(a, s);
  }
}

}  // namespace

size_t latent_attention_workspace(int64_t, int queries, int heads, int rank) {
  const size_t kn = rows_per_tile(queries * heads);
  return sm_count() * (2 * kn * (rank * sizeof(float) + sizeof(float2)) + sizeof(Cut));
}

cudaError_t launch_latent_attention(const LatentAttentionArgs& a, cudaStream_t s) {
  if (a.batch == 0) return cudaSuccess;
  return a.dtype == kF16 ? launch_rows<kF16>(a, s) : launch_rows<kBF16>(a, s);
}

}  // namespace exlr8
