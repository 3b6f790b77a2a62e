// Attention of many rows per sequence and key head over the 4-bit cache: chunks of prompts and whole prompts, on the tensor cores.
//
// A CTA (one per SM) walks its piece of the line of 128-position tiles.  A unit's up to 256 rows are two slots of 128, the M of an MMA:
//   S = Q K^T   tcgen05.mma kind::f16.  Keys are code * group scale, which f16 holds exactly; a row of q, scaled by a power of two, too (down
//               to 2^-29 of its largest).
//   P           softmax warps, four rows to a lane.  With x in units of log2 and references m (of the sum l) and n (of O) that follow a row's
//               largest score and its largest product of weight and value scale, l = sum 2^(x - m) and P = 2^(x - n + 5) * vscale, rounded to
//               f16, back into tensor memory over S.
//   O += P V    kind::f16, P from tensor memory, values as code * group scale in shared memory, exact again.
// Four converting warps, a thread per position, keep its key's and value's codes in registers while the stages in front are in use, so
// nothing but f16 tiles lies in shared memory.  The slots are out of step by half a tile: while the softmax warps of one work, the tensor
// core works for the other.  A unit of at most 128 rows takes turns: its even tiles are slot 0's, its odd ones slot 1's, and the sums are
// added up at the end.
//
// n comes from a bound, the row's largest score of the first tile times that tile's largest value scale.  That is near enough while the tile's
// scales are within a factor of 4 (the largest P is then 2^3 at least, and what f16 drops 2^-28 of it at most); a tile whose scales are
// further apart takes the products' own largest, as decoding does.  That reads the scores three times instead of once and takes the exponentials
// twice, and the value scales of a model's tokens seldom lie within a factor of 4 over 128 positions: the times below, of scales within a factor of 3, are
// then 1600 us (the prompt), 860 (the chunk with heads of 64), 910 (with heads of 128, 375), 240 (two chunks with a window, 139) and 130 (eight
// sequences of 1 to 250 new tokens, 80), whether the scales have a log-normal spread by factors of 2 or 4 or are those that the writing kernel
// leaves of normal vectors times 0.3 .. 1.3.  One scale far below the others costs its own tile only.
// Scores that are far apart let weights outgrow the reference, which are then done again: with a standard deviation of 4 instead of 1.5
// 1245 us (the prompt), 528, 598, 254 and 125, with 8 1366, 576, 664, 254 and 135.
//
// What bounds it is a slot's chain of scores, weights and product: a tile of 256 rows takes 4700 clocks, in which the exponentials' units work for
// 2048 and the tensor core for 2048 (heads of 128); leaving all exponentials out gains 9 %, seven of eight MMAs 6 %: half of the issue slots are
// empty, each slot waits for itself.  A tile of a unit that takes turns takes 3700: its conversion 2800, and loads that find as much on its way as
// the L1 beside 214 KB of shared memory holds.  A unit costs some 14000 clocks besides its tiles.  A prompt of 8192 tokens, 32 heads over 8:
// 647 to 660 us, 833 TFLOP/s and more of what is visible; 512 tokens behind 40000 positions with heads of 64: 328 to 338 us, 493 TFLOP/s
// and more (softmax work is twice that of heads of 128 per flop).
#include "kv4_chunk.cuh"
#include "stream_scratch.h"

namespace syfi {

namespace {

constexpr int kTile = 128;             // positions per tile: two pages
constexpr int kChunkRows = 256;
constexpr int kChunkThreads = 512;     // 8 softmax warps, 4 converting ones, then MMAs, planning, two idle ones
constexpr int kSoftmaxWarps = 8, kSoftmaxThreads = 256;
// What a unit counts besides its tiles, in tiles: by its clocks three, fitted five, which is flat around there.  With 3, 5 and 8: a prompt of 8192
// tokens 661, 647 and 670 us (its first pieces hold many short units), three of 1000 85, 84 and 88, two of 2500 with heads of 64 130, 131 and
// 138; two chunks with a window of 1024 141, 138 and 137, one of 2000 tokens with a window of 4096 202, 199 and 201; eight sequences of 1 to
// 250 new tokens 78, 75 and 73, twelve with heads of 64 89, 86 and 85.
constexpr int kChunkExtra = 5;
constexpr int kSlotRows = 128;         // units of at most so many rows use one slot for their even tiles and one for their odd ones
// (To the plan a tile of those is a tile like any other: it takes 3700 clocks, as its conversion is hidden behind nothing, and a tile of 256 rows 4700.
// Counted as half of one: eight sequences of 1 to 250 new tokens 84 us instead of 82.)
using ChunkPlan = Plan<kTile, kChunkRows, kChunkExtra>;
using ChunkCursor = Cursor<kTile, kChunkRows, kChunkExtra>;
constexpr int kScaleStages = 4;
constexpr int kStatusTimeout = 401;

// P is kept times 2^5 and may grow to 2^15 before the reference follows: a step of a row's reference stops its whole slot while O fades, and of
// 256 rows one or another took such a step in every other tile when P might grow by 2^5 only (512 tokens behind 40000 positions, scores of
// standard deviation 1.5: 618 us).
constexpr float kProductHeadroom = 5.0f;
constexpr float kProductGrowth = 9.0f;      // (where the reference is set from a bound that may be twice too low)
constexpr float kBlindGrowth = 1.0f;        // (where few positions gave it: 2^9 too low, it would not last)
constexpr float kNear = 0.25f;              // a tile's value scales are so near one another, or the products themselves are asked (both sides: at the top)
constexpr float kFarAbove = 60.0f;          // a row whose n lies so many octaves above m, because of a huge value, keeps its weights in units of m

template <int D>
struct ChunkShape {
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kTileBytes = kTile * D * 2;                // f16: [D / 64][128 rows][64], rows of 128 bytes, swizzled
  static constexpr int kQ = 0;                                    // [2 slots]
  static constexpr int kK = kQ + 2 * kTileBytes;
  static constexpr int kV = kK + kStages * kTileBytes;
  static constexpr int kScales = kV + kStages * kTileBytes;       // [K 128 f32][V 128 f32] per stage
  static constexpr int kHandOver = kScales + kScaleStages * 2 * kTile * 4;      // [4 warps][4][32 lanes] of four f32
  static constexpr int kSmem = 1024 + kHandOver + 4 * 4 * 32 * 16;
};

// A piece of a unit, as the planning warp describes it to the others.
struct Segment {
  int tile0, tiles;                    // tiles [tile0, tile0 + tiles) of the sequence's positions; no tiles: the piece is done
  int rows, row0;                      // rows [row0, row0 + rows) of the sequence's count * group
  int head, b, q_first;                // key head, sequence, its first row of q
  int base;                            // position of the sequence's first query
  int any_low, any_high, all_low, all_high;   // positions that any / all of the rows see
  int whole;                           // the unit lies in this piece alone
  int turns;                           // both slots work on rows 0 .. 127 and take turns at the tiles
  int first_part, last_part, first_slot;   // else: its Parts
};
__device__ __forceinline__ Parts parts_of(const Segment& g) { return {g.first_part, g.last_part, g.first_slot}; }
constexpr int kSegmentRing = 4;
constexpr int kSegmentReaders = 1 + 4 + kSoftmaxWarps;    // arrivals that free an entry: MMAs, converting and softmax warps

struct ChunkShared {
  Segment segment[kSegmentRing];
  uint64_t segment_full[kSegmentRing], segment_empty[kSegmentRing];
  uint64_t scale_full[kScaleStages], scale_empty[kScaleStages], k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t q_full[2], s_full[2], p_half[2], half_done[2], p_full[2], o_full[2], o_empty[2], idle;
  uint32_t tmem;
  int flags[kScaleStages];             // 1, 2: the tile's pages are there; 4: its value scales are near one another, none of them zero
  float largest[kScaleStages];         // of the value scales that any row sees
  float2 part[4];                      // largest and smallest of each converting warp's 32 positions
  int part_there[4];
  alignas(16) float4 end[2][128];      // [slot][row] m, l and n, at a segment's end
  float unit[256];                     // of each row: what a score is worth
  int2 bounds[2][128];                 // [slot][row]: the positions that it sees, counted from the segment's first tile
  int2 common[kSoftmaxWarps];          // the positions that all of a softmax warp's rows see
  volatile int abort_code;
  volatile uint32_t tiles_done;
  volatile int done;                   // every segment is
  int finished;                        // segments of this CTA whose results are written
};

// The CTA's piece of the line.
struct Piece {
  long long total, w1;
  int ctas, places;
};

// Waits ask only whether somebody gave up; the clock is the planning thread's, which has time.
__device__ __forceinline__ bool wait_for(ChunkShared& sh, uint64_t* bar, uint32_t parity) {
  while (!mbar_try_wait(bar, parity))
    if (sh.abort_code != 0) return false;
  return true;
}
// The same for warps that have to stay whole: a lane whose wait ran out goes on, and the warp asks for the abort code later.
__device__ __forceinline__ void wait_whole_warp(ChunkShared& sh, uint64_t* bar, uint32_t parity) { wait_for(sh, bar, parity); }

// A place in a ring of stages: its index, and the parity of its use.
template <int N>
struct Ring {
  int stage = 0;
  uint32_t parity = 0;
  __device__ void next() {
    if (++stage == N) {
      stage = 0;
      parity ^= 1u;
    }
  }
};

__device__ __forceinline__ void prefetch_l2(const void* p, int bytes) {      // both multiples of 16
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// ---------------------------------------------------------------- planning, and the clock (one thread)
struct Watch {
  long long limit, since;
  uint32_t seen;
  __device__ bool over(ChunkShared& sh) {
    const long long now = clock64();
    if (sh.tiles_done != seen) {
      seen = sh.tiles_done;
      since = now;
    } else if (now - since > limit) {
      sh.abort_code = kStatusTimeout;
    }
    return sh.abort_code != 0;
  }
};

template <int D>
__device__ __forceinline__ void plan_role(const AttentionArgs& a, const ChunkPlan& plan, const PlanShared& s_plan, ChunkShared& sh, const Piece& piece, long long wait_limit) {
  Watch watch = {wait_limit, clock64(), 0u};
  ChunkCursor at;
  at.start(plan, s_plan, piece.places);
  Ring<kSegmentRing> ring;
  while (true) {
    while (!mbar_try_wait(&sh.segment_empty[ring.stage], ring.parity ^ 1u))
      if (watch.over(sh)) return;
    Segment& g = sh.segment[ring.stage];
    const bool more = at.left > 0;
    const int here = more ? at.tiles_here() : 0;
    g.tiles = 0;
    if (more) {
      const int rows = at.rows(a.group), base = at.s.length - at.s.count, row0 = at.rt * kChunkRows;
      const int first = base + row0 / a.group, last = base + (row0 + rows - 1) / a.group;
      g.any_low = a.window > 0 ? max(first - a.window + 1, 0) : 0;
      g.any_high = last;
      g.tile0 = at.span.first + at.tile;
      g.tiles = here;
      g.turns = rows <= kSlotRows && g.tiles > 1;
      g.rows = rows;
      g.row0 = row0;
      g.head = at.head;
      g.b = at.b;
      g.q_first = at.s.first;
      g.base = base;
      g.all_low = a.window > 0 ? max(last - a.window + 1, 0) : 0;
      g.all_high = first;
      g.whole = here == at.span.tiles;
      const Parts parts(piece.total, piece.ctas, piece.w1 - at.left - at.tile, at.span.tiles);
      g.first_part = parts.first;
      g.last_part = parts.last;
      g.first_slot = parts.first_slot;
    }
    mbar_arrive(&sh.segment_full[ring.stage]);
    if (!more) break;
    // Its queries, for the softmax warps to find in L2: they ask for them only when the unit in front is done.
    for (int token = g.row0 / a.group; token <= (g.row0 + g.rows - 1) / a.group; ++token) {
      const int from = max(g.row0 - token * a.group, 0), to = min(g.row0 + g.rows - token * a.group, a.group);      // of the token's query heads
      prefetch_l2(a.q + (g.q_first + token) * a.q_stride + (g.head * a.group + from) * D, (to - from) * D * 2);
    }
    ring.next();
    at.advance(plan, here);
  }
  while (sh.done == 0 && !watch.over(sh)) __nanosleep(200);
}

// ---------------------------------------------------------------- MMAs (one thread)
template <int D>
__device__ __forceinline__ void mma_role(ChunkShared& sh, uint8_t* smem, uint32_t tmem) {
  using Shape = ChunkShape<D>;
  constexpr int kStages = Shape::kStages;
  const uint32_t qk_desc = umma_idesc_f16_m128(kTile), pv_desc = umma_idesc_f16_m128_n_major(D);
  const uint64_t q_desc = umma_smem_desc_sw128(smem_u32(smem + Shape::kQ));
  const uint64_t v_desc = umma_smem_desc_n_major_sw128(smem_u32(smem + Shape::kV), kTile * 128);
  const uint32_t q0 = static_cast<uint32_t>(q_desc), k0 = q0 + (Shape::kK - Shape::kQ) / 16, qk_hi = static_cast<uint32_t>(q_desc >> 32);
  const uint32_t v0 = static_cast<uint32_t>(v_desc), v_hi = static_cast<uint32_t>(v_desc >> 32);
  auto scores = [&](int slot, int q_slot, int stage) {
    const uint32_t k = k0 + stage * (Shape::kTileBytes / 16), q = q0 + q_slot * (Shape::kTileBytes / 16), to = tmem + slot * 128;
#pragma unroll
    for (int step = 0; step < D / 16; ++step) {
      const uint32_t at = step / 4 * (kTile * 128 / 16) + step % 4 * 2;
      umma_f16_words(to, q + at, k + at, qk_hi, qk_desc, step > 0 ? 1u : 0u);
    }
    umma_commit(&sh.s_full[slot]);
  };
  auto values = [&](int slot, int stage, int half, uint32_t add) {
    const uint32_t v = v0 + stage * (Shape::kTileBytes / 16), p = tmem + slot * 128;
#pragma unroll
    for (int i = 0; i < kTile / 32; ++i) {
      const int step = half * (kTile / 32) + i;
      umma_f16_ts_words(p + 256, p + 8 * step, v + 128 * step, v_hi, pv_desc, step == 0 ? add : 1u);
    }
  };
  Ring<kSegmentRing> segments;
  Ring<kStages> keys, vals;
  uint32_t tile_parity = 0, segment_parity = 0;    // bit s: of slot s
  // P of the slot's tile, in two halves, times its values
  auto product = [&](int s, int stage, uint32_t add) {
    const uint32_t parity = tile_parity >> s & 1u;
    tile_parity ^= 1u << s;
    if (!wait_for(sh, &sh.p_half[s], parity)) return false;
    tc_fence_after();
    values(s, stage, 0, add);
    umma_commit(&sh.half_done[s]);
    if (!wait_for(sh, &sh.p_full[s], parity)) return false;
    tc_fence_after();
    values(s, stage, 1, 1u);
    return true;
  };
  while (true) {
    if (!wait_for(sh, &sh.segment_full[segments.stage], segments.parity)) return;
    const Segment& g = sh.segment[segments.stage];
    const int n = g.tiles, turns = g.turns, slots = turns || g.rows > kSlotRows ? 2 : 1;
    if (n == 0) return;
    mbar_arrive(&sh.segment_empty[segments.stage]);
    segments.next();
    for (int s = 0; s < slots; ++s)
      if (!wait_for(sh, &sh.q_full[s], segment_parity >> s & 1u)) return;
    // A slot's scores of its next tile follow its values' product, which reads the weights in their place.
    if (turns) {                             // tile j in slot j % 2
      for (int j = 0; j < 2; ++j) {
        if (!wait_for(sh, &sh.k_full[keys.stage], keys.parity)) return;
        tc_fence_after();
        scores(j, 0, keys.stage);
        umma_commit(&sh.k_empty[keys.stage]);
        keys.next();
      }
      for (int j = 0; j < n; ++j) {
        const int s = j & 1;
        const bool more = j + 2 < n;
        if (j < 2 && !wait_for(sh, &sh.o_empty[s], (segment_parity >> s & 1u) ^ 1u)) return;
        if (!wait_for(sh, &sh.v_full[vals.stage], vals.parity)) return;
        if (!product(s, vals.stage, j < 2 ? 0u : 1u)) return;
        umma_commit(&sh.v_empty[vals.stage]);
        vals.next();
        if (more) {
          if (!wait_for(sh, &sh.k_full[keys.stage], keys.parity)) return;
          tc_fence_after();
          scores(s, 0, keys.stage);
          umma_commit(&sh.k_empty[keys.stage]);
          keys.next();
        } else {
          umma_commit(&sh.o_full[s]);
        }
      }
      segment_parity ^= 3u;
      continue;
    }
    if (!wait_for(sh, &sh.k_full[keys.stage], keys.parity)) return;
    tc_fence_after();
    for (int s = 0; s < slots; ++s) scores(s, s, keys.stage);
    umma_commit(&sh.k_empty[keys.stage]);
    keys.next();
    for (int j = 0; j < n; ++j) {
      const bool more = j + 1 < n;
      if (more && !wait_for(sh, &sh.k_full[keys.stage], keys.parity)) return;
      if (!wait_for(sh, &sh.v_full[vals.stage], vals.parity)) return;
#pragma unroll 1
      for (int s = 0; s < slots; ++s) {
        if (j == 0 && !wait_for(sh, &sh.o_empty[s], (segment_parity >> s & 1u) ^ 1u)) return;
        if (!product(s, vals.stage, j > 0 ? 1u : 0u)) return;
        if (s + 1 == slots) umma_commit(&sh.v_empty[vals.stage]);
        if (more) scores(s, s, keys.stage);
        else umma_commit(&sh.o_full[s]);
      }
      vals.next();
      if (more) {
        umma_commit(&sh.k_empty[keys.stage]);
        keys.next();
      }
    }
    segment_parity ^= slots == 2 ? 3u : 1u;
  }
}

// ---------------------------------------------------------------- codes to f16, a thread per position (four warps)
// 32 bytes that are read once.  Two loads, since a cache and its pages begin at any multiple of 16 bytes.  (One of 32, where they begin at multiples
// of that, is no faster: 512 tokens behind 40000 positions 343 us by one and 342 by two, with heads of 128 379 and 374; and in lines that
// stay in the L1 383.)
__device__ __forceinline__ void ld_global_32(const void* p, uint4& a, uint4& b) {
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w) : "l"(p));
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4 + 16];" : "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "l"(p));
}
__device__ __forceinline__ void st_shared_16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// A row of codes and its scales on their way from the cache.
template <int D>
struct RawRow {
  uint4 codes[D / 32];
  uint32_t groups[D / 64];
  float scale;
  __device__ __forceinline__ void ask(const uint8_t* block, int at) {
#pragma unroll
    for (int p = 0; p < D / 64; ++p) ld_global_32(block + p * kKv4Plane + at * 32, codes[2 * p], codes[2 * p + 1]);
    const uint32_t* const from = reinterpret_cast<const uint32_t*>(block + Kv4Block<D>::kGroups + at * (D / kKv4Group));
    if constexpr (D == 128) {
      const uint2 g = __ldg(reinterpret_cast<const uint2*>(from));
      groups[0] = g.x;
      groups[1] = g.y;
    } else {
      groups[0] = __ldg(from);
    }
    scale = __ldg(reinterpret_cast<const float*>(block + Kv4Block<D>::kScales) + at);
  }
  // code * group scale as f16 into a tile's row (`to`: where its first 16 bytes lie, in rows of 128 that are swizzled)
  __device__ __forceinline__ void put(uint32_t to) const {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const uint32_t w[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
      // two groups of 16 dimensions, 8 in a word
      const uint32_t both = e4m3x2_to_half2(groups[i / 2] >> (16 * (i % 2)));
      const uint32_t scale[2] = {__byte_perm(both, both, 0x1010), __byte_perm(both, both, 0x3232)};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        st_shared_16((to ^ (i % 2 * 4 + k) * 16) + i / 2 * (kTile * 128), hmul2_bits(e2m1x2_to_half2<0>(w[k]), scale[k / 2]), hmul2_bits(e2m1x2_to_half2<1>(w[k]), scale[k / 2]),
                     hmul2_bits(e2m1x2_to_half2<2>(w[k]), scale[k / 2]), hmul2_bits(e2m1x2_to_half2<3>(w[k]), scale[k / 2]));
      }
    }
  }
};

// A barrier of the converting warps that tells all of them whether any thread's `p` holds.
__device__ __forceinline__ bool converters_any(bool p) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 7, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(p))
      : "memory");
  return any != 0u;
}

template <int D>
__device__ __forceinline__ void convert_role(const AttentionArgs& a, ChunkShared& sh, uint8_t* smem) {
  using Shape = ChunkShape<D>;
  constexpr int kStages = Shape::kStages;
  const int t = threadIdx.x % 128, lane = threadIdx.x % 32, warp = t / 32, page_of = t / kKvPage, at = t % kKvPage;
  Ring<kSegmentRing> segments;           // of the tile to ask for
  Ring<kScaleStages> scales;
  Ring<kStages> tiles;
  // The walk of the loads: a tile's rows are asked for as soon as those of the tile in front are converted, its table entry two tiles
  // earlier, so that neither is waited for.
  struct Ahead {
    int entry;                           // a page of the cache, or none
    int head_flags;                      // key head * 4, 2: any row sees the position, 1: all rows see the tile
  };
  int next_tile = 0, left = 0;
  auto look_ahead = [&](Ahead& e) -> bool {      // whole warp; false behind the last tile
    const Segment& g = sh.segment[segments.stage];
    if (left == 0) {
      wait_whole_warp(sh, &sh.segment_full[segments.stage], segments.parity);
      __syncwarp();
      left = g.tiles;                    // (behind a failure an older segment's, or none: the same for the four warps)
      if (left == 0) return false;
      next_tile = g.tile0;
    }
    const int page = 2 * next_tile + page_of, first = next_tile * kTile;
    e.entry = page < a.batch.max_pages && page * kKvPage <= g.any_high && (page + 1) * kKvPage > g.any_low
                  ? __ldg(a.batch.block_table + static_cast<long long>(g.b) * a.batch.max_pages + page) : -1;
    e.head_flags = g.head * 4 + (first + t >= g.any_low && first + t <= g.any_high ? 2 : 0) + (first >= g.all_low && first + kTile - 1 <= g.all_high ? 1 : 0);
    ++next_tile;
    if (--left == 0) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.segment_empty[segments.stage]);
      segments.next();
    }
    return true;
  };
  auto is_there = [&](const Ahead& e) { return e.entry >= 0 && e.entry < a.cache.num_pages; };
  const uint32_t row = smem_u32(smem) + Shape::kK + t * 128 + (t & 7) * 16;      // in the keys' first stage
  RawRow<D> key, value;
  Ahead now, next, behind;               // of the rows in registers, and of the two tiles that follow
  bool here = look_ahead(now);
  if (here && is_there(now)) {
    key.ask(kv4_block<D>(a.cache, now.entry, 0, now.head_flags >> 2), at);
    value.ask(kv4_block<D>(a.cache, now.entry, 1, now.head_flags >> 2), at);
  }
  bool more = here && look_ahead(next);
  while (here) {
    const bool more_behind = more && look_ahead(behind), there = is_there(now);
    wait_whole_warp(sh, &sh.k_empty[tiles.stage], tiles.parity ^ 1u);
    __syncwarp();
    if (there) key.put(row + tiles.stage * Shape::kTileBytes);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.k_full[tiles.stage]);
    float ks = there ? key.scale : 0.0f;
    if (more && is_there(next)) key.ask(kv4_block<D>(a.cache, next.entry, 0, next.head_flags >> 2), at);
    // What a row does not see must not reach its sums, and zero times NaN is NaN: values of positions that no row sees become zeros, and
    // where some rows see a value that is not finite, the NaN goes by way of its score to those rows alone.
    float vs = there ? value.scale : 1.0f;
    bool bad = !(fabsf(vs) <= 3.402823466e38f);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) bad |= there && (((value.groups[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0u;
    const bool valid = there && (now.head_flags & 2) && ((now.head_flags & 1) || !bad);
    if (bad || !(fabsf(ks) <= 3.402823466e38f)) ks = __int_as_float(0x7fffffff);
    if (!valid) vs = 1.0f;
    const unsigned bits = __float_as_uint(vs);
    const bool counts = valid && bits < 0x7f800000u;
    const unsigned high = __reduce_max_sync(0xffffffffu, counts ? bits : 0u), low = __reduce_min_sync(0xffffffffu, counts ? bits : 0x7f800000u);
    wait_whole_warp(sh, &sh.scale_empty[scales.stage], scales.parity ^ 1u);
    __syncwarp();
    float* const to = reinterpret_cast<float*>(smem + Shape::kScales) + scales.stage * 2 * kTile;
    to[t] = ks;
    to[kTile + t] = vs;
    if (lane == 0) {
      sh.part[warp] = make_float2(__uint_as_float(high), __uint_as_float(low));
      sh.part_there[warp] = there;
    }
    named_bar_sync(7, 128);
    if (t == 0) {
      float largest = 0.0f, smallest = INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        largest = fmaxf(largest, sh.part[w].x);
        smallest = fminf(smallest, sh.part[w].y);
      }
      // (the weights' sum, in units of n, is in f32's range)
      const bool near = smallest >= kNear * largest && largest >= 1e-18f && largest <= 1e18f;
      sh.largest[scales.stage] = largest;
      sh.flags[scales.stage] = (sh.part_there[0] ? 1 : 0) | (sh.part_there[2] ? 2 : 0) | (near ? 4 : 0);
      mbar_arrive(&sh.scale_full[scales.stage]);
    }
    __syncwarp();
    const bool gone = converters_any(sh.abort_code != 0);     // (and the parts are read)
    scales.next();
    wait_whole_warp(sh, &sh.v_empty[tiles.stage], tiles.parity ^ 1u);
    __syncwarp();
    const uint32_t to_row = row + (Shape::kV - Shape::kK) + tiles.stage * Shape::kTileBytes;
    if (valid) {
      value.put(to_row);
    } else {
#pragma unroll 1
      for (int chunk = 0; chunk < D / 8; ++chunk) st_shared_16((to_row ^ chunk % 8 * 16) + chunk / 8 * (kTile * 128), 0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.v_full[tiles.stage]);
    tiles.next();
    if (more && is_there(next)) value.ask(kv4_block<D>(a.cache, next.entry, 1, next.head_flags >> 2), at);
    if (gone) return;                  // all four together
    here = more;
    now = next;
    more = more_behind;
    next = behind;
  }
}

// ---------------------------------------------------------------- softmax (eight warps, four to a slot, 32 rows each)
// A lane has four rows, 8 i + lane / 4, and of every eight positions two, 2 (lane % 4) and the next: the accumulator's layout of an m16n8 MMA,
// which tensor memory's 16x256b loads give.  So a scale that is read serves four rows; with a row to a lane, the scales' 64 reads of 16 bytes a
// tile and warp alone took the shared memory's port for 2000 clocks of a tile.
__device__ __forceinline__ uint64_t ld_shared_pair(uint32_t at) {
  uint64_t v;
  asm volatile("ld.shared.u64 %0, [%1];" : "=l"(v) : "r"(at));
  return v;
}

// What the softmax of a tile works with.
struct TileRows {
  uint32_t t_s;                        // tensor memory: scores (weights over their first half); the sums lie 256 columns on
  uint32_t scales;                     // shared memory: this lane's first of 128 scales of keys, then of values
  const int2* bounds;                  // shared memory: lowest and highest position that each of the slots' rows sees
  int offset;                          // of the tile in those
  bool masked, there0, there1;         // whether any of that matters for the warp's rows; the tile's pages
  bool near;                           // the tile's value scales are near one another
  float unit[4];                       // what a score is worth
};
__device__ __forceinline__ int2 row_bounds(const TileRows& r, int row) {
  const int2 v = r.bounds[threadIdx.x / 32 * 32 + threadIdx.x % 32 / 4 + 8 * row];
  return make_int2(v.x - r.offset, v.y - r.offset);
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}

// 64 scores of this lane's four rows, from position 64 h of the tile on
__device__ __forceinline__ void load_scores(const TileRows& r, int h, uint32_t (&s)[2][32]) {
  tmem_ld_16x256b(r.t_s + 64 * h, s[0]);
  tmem_ld_16x256b(r.t_s + 64 * h + (16u << 16), s[1]);
}
__device__ __forceinline__ void scores_landed(uint32_t (&s)[2][32]) {
  tmem_ld_wait_for(s[0]);
  tmem_landed(s[1]);
}

// O of the warp's rows times `fade`.
template <int D>
__device__ __forceinline__ void rescale_sums(uint32_t t_o, const float (&fade)[4]) {
#pragma unroll 1
  for (int k = 0; k < 2 * (D / 64); ++k) {
    const uint32_t at = t_o + (k & 1 ? 16u << 16 : 0u) + k / 2 * 64;
    uint32_t o[32];
    tmem_ld_16x256b(at, o);
    tmem_ld_wait_for(o);
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * (k & 1 ? fade[2 + e / 2 % 2] : fade[e / 2 % 2]));
    tmem_st_16x256b(at, o);
  }
  tmem_st_wait();
}

// A score is S times (its key's scale times its row's unit), here and below: a row of q is kept at most 2^120 times its size, so that S times the
// key's scale alone can run over where tiny queries meet huge keys, although the score is an ordinary number.

// The rows' largest scores of 64 positions.
template <bool MASKED>
__device__ __forceinline__ void largest_scores(const TileRows& r, int h, const uint32_t (&s)[2][32], float (&top)[4]) {
  const int column = 64 * h + threadIdx.x % 4 * 2;
  const bool there = h == 0 ? r.there0 : r.there1;
#pragma unroll
  for (int row = 0; row < 4; ++row) {
    const int2 see = MASKED ? row_bounds(r, row) : make_int2(0, 0);
    const uint64_t unit = f32x2_pack(r.unit[row], r.unit[row]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint64_t worth = f32x2_mul(ld_shared_pair(r.scales + 4 * (64 * h + 8 * i)), unit);
      float x0, x1;
      f32x2_unpack(f32x2_mul(f32x2_pack_bits(s[row / 2][4 * i + 2 * (row % 2)], s[row / 2][4 * i + 2 * (row % 2) + 1]), worth), x0, x1);
      const int at = column + 8 * i;
      if (!MASKED || (there && at >= see.x && at <= see.y)) top[row] = fmaxf(top[row], x0);
      if (!MASKED || (there && at + 1 >= see.x && at + 1 <= see.y)) top[row] = fmaxf(top[row], x1);
    }
  }
}

// Weights of 64 positions, times the values' scales, as pairs of f16, and their sums; returns whether one does not fit (of all four rows).
// GENERAL: positions that a row does not see, and products times `factor`.
template <bool GENERAL>
__device__ __forceinline__ bool half_weights(const TileRows& r, int h, const uint32_t (&s)[2][32], const float (&shift)[4], const float (&factor)[4], float (&total)[4],
                                             uint32_t (&p)[2][16]) {
  uint32_t most[2] = {0u, 0u};
  uint64_t sums[4];
  int2 see[4];
#pragma unroll
  for (int row = 0; row < 4; ++row) {
    sums[row] = 0ull;
    see[row] = make_int2(0, 0);
    if (GENERAL) {
      see[row] = row_bounds(r, row);
      if (!(h == 0 ? r.there0 : r.there1)) see[row].y = -1;
    }
  }
  const int column = 64 * h + threadIdx.x % 4 * 2;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint64_t ks = ld_shared_pair(r.scales + 4 * (64 * h + 8 * i)), vs = ld_shared_pair(r.scales + 4 * (kTile + 64 * h + 8 * i));
#pragma unroll
    for (int row = 0; row < 4; ++row) {
      const uint64_t worth = f32x2_mul(ks, f32x2_pack(r.unit[row], r.unit[row]));
      float x0, x1;
      f32x2_unpack(f32x2_fma(f32x2_pack_bits(s[row / 2][4 * i + 2 * (row % 2)], s[row / 2][4 * i + 2 * (row % 2) + 1]), worth, f32x2_pack(shift[row], shift[row])), x0, x1);
      x0 = ex2(x0);
      x1 = ex2(x1);
      if (GENERAL) {
        const int at = column + 8 * i;
        x0 = at >= see[row].x && at <= see[row].y ? x0 : 0.0f;
        x1 = at + 1 >= see[row].x && at + 1 <= see[row].y ? x1 : 0.0f;
      }
      uint64_t w = f32x2_pack(x0, x1);
      sums[row] = f32x2_add(sums[row], w);
      w = f32x2_mul(w, vs);
      if (GENERAL) w = f32x2_mul(w, f32x2_pack(factor[row], factor[row]));
      f32x2_unpack(w, x0, x1);
      p[row / 2][2 * i + row % 2] = pack_half2(x0, x1);
      most[row / 2] = hmax2_bits(most[row / 2], p[row / 2][2 * i + row % 2]);
    }
  }
#pragma unroll
  for (int row = 0; row < 4; ++row) {
    float a0, a1;
    f32x2_unpack(sums[row], a0, a1);
    total[row] = a0 + a1;
  }
  const uint32_t top = hmax2_bits(most[0], most[1]);
  return (top & 0xffffu) > 0x7800u || top >> 16 > 0x7800u;      // 2^15 (the maximum of two is no NaN unless all are)
}

// The largest product of a weight, in units of `shift`, and its value's scale in 64 positions.
__device__ __forceinline__ void largest_products(const TileRows& r, int h, const uint32_t (&s)[2][32], const float (&shift)[4], float (&most)[4]) {
  const int column = 64 * h + threadIdx.x % 4 * 2;
  const bool there = h == 0 ? r.there0 : r.there1;
#pragma unroll
  for (int row = 0; row < 4; ++row) {
    const int2 see = row_bounds(r, row);
    const uint64_t unit = f32x2_pack(r.unit[row], r.unit[row]), from = f32x2_pack(shift[row], shift[row]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint64_t worth = f32x2_mul(ld_shared_pair(r.scales + 4 * (64 * h + 8 * i)), unit);
      float x0, x1, v0, v1;
      f32x2_unpack(f32x2_fma(f32x2_pack_bits(s[row / 2][4 * i + 2 * (row % 2)], s[row / 2][4 * i + 2 * (row % 2) + 1]), worth, from), x0, x1);
      f32x2_unpack(ld_shared_pair(r.scales + 4 * (kTile + 64 * h + 8 * i)), v0, v1);
      const int at = column + 8 * i;
      if (there && at >= see.x && at <= see.y) most[row] = fmaxf(most[row], ex2(x0) * v0);
      if (there && at + 1 >= see.x && at + 1 <= see.y) most[row] = fmaxf(most[row], ex2(x1) * v1);
    }
  }
}

// References for a tile from its scores themselves: m, with l in its units, and n from the bound, or with `products` from the products' own
// largest.  fade: what O becomes smaller by.
__device__ __forceinline__ void set_references(const TileRows& r, float largest, bool products, float (&m)[4], float (&n)[4], float (&l)[4], float (&fade)[4]) {
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, bound[4];
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    uint32_t s[2][32];
    load_scores(r, h, s);
    scores_landed(s);
    if (r.masked) largest_scores<true>(r, h, s, top);
    else largest_scores<false>(r, h, s, top);
  }
#pragma unroll
  for (int row = 0; row < 4; ++row) {
    top[row] = quad_max(top[row]);
    if (top[row] > m[row]) {
      l[row] *= ex2(m[row] - top[row]);        // (0 for a row that had seen nothing)
      m[row] = top[row];
    }
    bound[row] = top[row] + lg2(largest);
  }
  if (products) {
    float most[4] = {}, shift[4];
#pragma unroll
    for (int row = 0; row < 4; ++row) shift[row] = -finite_or_zero(m[row]);
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      uint32_t s[2][32];
      load_scores(r, h, s);
      scores_landed(s);
      largest_products(r, h, s, shift, most);
    }
#pragma unroll
    for (int row = 0; row < 4; ++row) bound[row] = m[row] + fmaxf(lg2(quad_max(most[row])), -90.0f);      // (never further behind: a value may be zero)
  }
#pragma unroll
  for (int row = 0; row < 4; ++row) {
    fade[row] = 1.0f;
    if (bound[row] > n[row] + (products ? kProductGrowth : kBlindGrowth)) {
      fade[row] = ex2(n[row] - bound[row]);
      n[row] = bound[row];
    }
  }
}

// The weights of a tile, half of it at a time: into tensor memory over scores that are used up.  A reference n stays what it is unless a weight
// does not fit, which hardly ever happens; then the row's O and l fade, and the half is done again.  GENERAL: rows that do not see every
// position, and `careful`: weights in units of m first, for tiles whose value scales are far apart.
template <int D, bool GENERAL>
__device__ __forceinline__ void tile_weights(ChunkShared& sh, const TileRows& r, int slot, uint32_t tile_parity, bool first, bool careful, float largest,
                                             float (&m)[4], float (&n)[4], float (&l)[4]) {
  const int lane = threadIdx.x % 32;
  float shift[4], factor[4], worth[4];   // worth: of this tile's weights in the sum (a step of the references leaves it)
#pragma unroll
  for (int row = 0; row < 4; ++row) {
    shift[row] = GENERAL && careful ? -finite_or_zero(m[row]) : kProductHeadroom - finite_or_zero(n[row]);
    factor[row] = !(GENERAL && careful) ? 1.0f : m[row] != -INFINITY && n[row] != -INFINITY ? ex2(m[row] - n[row] + kProductHeadroom) : 0.0f;
    worth[row] = GENERAL && careful ? 1.0f : ex2(-shift[row] - finite_or_zero(m[row]));
  }
  uint32_t s[2][32];
  load_scores(r, 0, s);
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    uint32_t p[2][16];
    float total[4];
    for (bool again = false;; again = true) {
      scores_landed(s);
      const bool over = half_weights<GENERAL>(r, h, s, shift, factor, total, p);
      // (in units of m nothing can be over that was finite)
      if (__builtin_expect(!__any_sync(0xffffffffu, over), 1) || again || (GENERAL && careful)) break;
      load_scores(r, h, s);
      scores_landed(s);
      float highest[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, fade[4];
      largest_scores<true>(r, h, s, highest);
#pragma unroll
      for (int row = 0; row < 4; ++row) {
        const float bound = quad_max(highest[row]) + shift[row] + lg2(largest), up = bound > 15.0f ? bound - kProductHeadroom : 0.0f;
        fade[row] = ex2(-up);
        n[row] += up;
        shift[row] -= up;
        m[row] += up;                  // (the sum's reference goes along, so that the two stay near)
        l[row] *= fade[row];
      }
      if (h == 1) {                    // the first half's product is on its way
        wait_whole_warp(sh, &sh.half_done[slot], tile_parity);
        __syncwarp();
        tc_fence_after();
      }
      if (!first || h == 1) rescale_sums<D>(r.t_s + 256, fade);
      load_scores(r, h, s);
    }
    if (h == 0) load_scores(r, 1, s);
    tmem_st_16x128b(r.t_s + 32 * h, p[0]);
    tmem_st_16x128b(r.t_s + 32 * h + (16u << 16), p[1]);
#pragma unroll
    for (int row = 0; row < 4; ++row) l[row] = fmaf(total[row], worth[row], l[row]);
    tmem_st_wait();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(h == 0 ? &sh.p_half[slot] : &sh.p_full[slot]);
  }
}

// What the warp's rows need before a tile's weights: nothing; references, because a row has none (kBlind, as at the start) or one from fewer than
// kEnough positions; or weights in units of m, because a row's n lies far above it (kFar).  (At a window's lower edge a row may see a few
// positions of its first tile, and of 256 rows one or another then had weights 2^10 larger in a later tile, done again at 5000 clocks and more.)
constexpr int kSettled = 0, kBlind = 1, kFar = 2;
constexpr int kEnough = 32;

// A tile of the warp's rows: scores from tensor memory, weights back into it; the rows' references m and n and this lane's part of their sums l.
template <int D>
__device__ __forceinline__ void softmax_tile(ChunkShared& sh, const TileRows& r, int slot, int stage, uint32_t tile_parity, bool first, int& settled, float (&m)[4],
                                             float (&n)[4], float (&l)[4]) {
  const float largest = sh.largest[stage];
  const bool careful = !r.near || settled == kFar;
  wait_whole_warp(sh, &sh.s_full[slot], tile_parity);
  __syncwarp();
  tc_fence_after();
  if (careful || settled != kSettled) {
    float fade[4];
    set_references(r, largest, careful, m, n, l, fade);
    if (!first && __any_sync(0xffffffffu, fade[0] != 1.0f || fade[1] != 1.0f || fade[2] != 1.0f || fade[3] != 1.0f)) rescale_sums<D>(r.t_s + 256, fade);
  }
  if (__builtin_expect(careful || r.masked, 0)) tile_weights<D, true>(sh, r, slot, tile_parity, first, careful, largest, m, n, l);
  else tile_weights<D, false>(sh, r, slot, tile_parity, first, false, largest, m, n, l);
  if (careful || settled != kSettled) {        // (neither far nor blind for a row that is not finite; steps of the references leave n - m)
    bool far = false, blind = false;
#pragma unroll
    for (int row = 0; row < 4; ++row) {
      far |= n[row] - m[row] > kFarAbove;
      blind |= n[row] == -INFINITY && l[row] == l[row];
      if (r.masked) {
        const int2 see = row_bounds(r, row);
        blind |= see.y >= kTile - 1 && see.x > kTile - kEnough;
      }
    }
    settled = __any_sync(0xffffffffu, far) ? kFar : __any_sync(0xffffffffu, blind) ? kBlind : kSettled;
  }
}

// The warp's 32 rows of q (of which `rows` are there; mine: where this lane's row begins in q) as f16 times 2^k each, the row's largest at
// 2^14 .. 2^15, into rows row0 and on of a tile.  Four lanes have a row, which takes two shuffles for its largest and the exponent's arithmetic
// for eight rows at a time; each second row starts with its other half, so that stores hit all banks.  units: what a score of each row is worth.
template <int D>
__device__ __forceinline__ void put_queries(const __nv_bfloat16* q, long long mine, float scale_log2, int rows, uint8_t* tile, int row0, float* units) {
  constexpr int kChunks = D / 32;          // of eight dimensions, a lane's
  const int lane = threadIdx.x % 32, part = lane % 4;
#pragma unroll 2
  for (int at = 0; at < 32; at += 8) {
    const int row = at + lane / 4, in_tile = row0 + row;
    const uint4* const from = reinterpret_cast<const uint4*>(q + __shfl_sync(0xffffffffu, mine, row)) + part;
    uint4 raw[kChunks];
    uint32_t most = 0u;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) raw[j] = row < rows ? __ldg(from + 4 * (j ^ (row & 1))) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      most = __vmaxu2(__vmaxu2(most, raw[j].x & 0x7fff7fffu), raw[j].y & 0x7fff7fffu);
      most = __vmaxu2(__vmaxu2(most, raw[j].z & 0x7fff7fffu), raw[j].w & 0x7fff7fffu);
    }
    most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const unsigned top = max(most & 0xffffu, most >> 16);
    const int k = top == 0u ? 0 : min(14 - (static_cast<int>(top >> 7) - 127), 120);
    const float up = copysignf(__int_as_float((k + 127) << 23), scale_log2);
    const uint64_t ups = f32x2_pack(up, up);
    // (a row that is not finite is NaN throughout, so that the mask takes its scores out like any other's)
    const uint32_t spoilt = top >= 0x7f80u ? 0x7fff7fffu : 0u;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
      uint32_t h[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x0, x1;
        f32x2_unpack(f32x2_mul(f32x2_pack_bits(w[e] << 16, w[e] & 0xffff0000u), ups), x0, x1);
        h[e] = pack_half2(x0, x1) | spoilt;
      }
      const int chunk = 4 * (j ^ (row & 1)) + part;
      *reinterpret_cast<uint4*>(tile + chunk / 8 * (kTile * 128) + in_tile * 128 + ((chunk % 8 ^ (in_tile & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
    }
    if (part == 0) units[row] = fabsf(scale_log2) * __int_as_float((127 - k) << 23);
  }
}

// A barrier of the softmax warps that tells all of them whether any thread's `p` holds.
__device__ __forceinline__ bool softmax_bar_any(bool p) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(p))
      : "memory");
  return any != 0u;
}

// Adds up a split unit's parts, kept by dimension ([part][D / 4][rows][4], then [part][rows] of (m, l, n, -)): a thread has a row and sixteen of
// its dimensions.
template <int D>
__device__ __forceinline__ void join_columns(const AttentionArgs& a, int q_first, int unit_row0, int head, int rows, int ctas, const Parts& parts, int thread, int threads) {
  const float4* const stats = reinterpret_cast<const float4*>(a.partial + 2ll * ctas * kChunkRows * D);
  const float4* const sums = reinterpret_cast<const float4*>(a.partial);
  const int across = (rows + 31) / 32 * 32;      // (whole warps of neighbouring rows: the join of a unit of 4 rows 2 us instead of 10, of 256 rows 8)
  for (int i = thread; i < across * (D / 16); i += threads) {
    const int row = i % across, d16 = i / across;
    if (row >= rows) continue;
    float m = -INFINITY, n = -INFINITY, l = 0.0f, o[16] = {};
#pragma unroll 2
    for (int c = parts.first; c <= parts.last; ++c) {
      const long long slot = parts.slot(c);
      const float4 st = __ldcg(stats + slot * kChunkRows + row);
      float4 p[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) p[k] = __ldcg(sums + (slot * (D / 4) + 4 * d16 + k) * kChunkRows + row);
      const float m_new = fmaxf(m, st.x), m_ref = finite_or_zero(m_new), n_new = fmaxf(n, st.z), n_ref = finite_or_zero(n_new);
      l = l * ex2(m - m_ref) + st.y * ex2(st.x - m_ref);
      const float f = ex2(n - n_ref), w = ex2(st.z - n_ref);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        o[4 * k] = o[4 * k] * f + p[k].x * w;
        o[4 * k + 1] = o[4 * k + 1] * f + p[k].y * w;
        o[4 * k + 2] = o[4 * k + 2] * f + p[k].z * w;
        o[4 * k + 3] = o[4 * k + 3] * f + p[k].w * w;
      }
      m = m_new;
      n = n_new;
    }
    const float f = l == 0.0f || n == -INFINITY ? 0.0f : ex2(n - finite_or_zero(m) - kProductHeadroom) / l;
    const int r = unit_row0 + row;
    uint4* const to = reinterpret_cast<uint4*>(a.out + (q_first + r / a.group) * a.out_stride + (head * a.group + r % a.group) * D + 16 * d16);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(o[8 * h + 2 * e] * f, o[8 * h + 2 * e + 1] * f);
        w[e] = *reinterpret_cast<const uint32_t*>(&b);
      }
      to[h] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// The thread's number, in a form from which nothing is computed ahead of a loop: what a segment's ends need would take the tiles' registers, and
// a register of theirs in local memory costs 600 clocks a use (the L1 is small beside this much shared memory).
__device__ __forceinline__ int thread_here() {
  int t = threadIdx.x;
  asm volatile("" : "+r"(t));
  return t;
}

template <int D>
__device__ __forceinline__ void softmax_role(const AttentionArgs& a, ChunkShared& sh, PlanShared& s_plan, uint8_t* smem, const Piece& piece) {
  using Shape = ChunkShape<D>;
  // warps 0-3: slot 0, 4-7: slot 1
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, slot = warp / 4;
  const uint32_t scales0 = smem_u32(smem) + Shape::kScales;
  static_assert(kSegmentRing == 4 && kScaleStages == 4, "stage and parity are bits of a counter");
  uint32_t segment = 0, tile = 0, own = 0;       // segments and tiles so far; parities of this slot's tiles (bit 0) and segments (bit 1)
  // A thread's row of a unit (rows beyond the last copy its bounds), and where it lies.
  auto row_of = [&](const Segment& g, int thread) { return g.turns ? thread % 128 : thread; };
  auto token_of = [&](const Segment& g, int row, int& column) {
    const int at = g.row0 + min(row, g.rows - 1), token = at / a.group;
    column = (g.head * a.group + at - token * a.group) * D;
    return token;
  };
  auto is_active = [&](const Segment& g, int slot) { return g.turns || g.rows > slot * kSlotRows; };
  // What a segment's tiles need of its rows: their bounds, and q in shared memory, where the MMAs of the one in front no longer read.
  auto begin = [&](const Segment& g) {
    const int thread = thread_here(), warp = thread / 32, lane = thread % 32, slot = warp / 4, in_slot = thread % 128;
    int column;
    const int token = token_of(g, row_of(g, thread), column), high = g.base + token - g.tile0 * kTile;
    const int low = a.window > 0 ? max(g.base + token - a.window + 1, 0) - g.tile0 * kTile : -g.tile0 * kTile;
    sh.bounds[slot][in_slot] = make_int2(low, high);      // counted from the segment's first tile
    const int highest_low = __reduce_max_sync(0xffffffffu, low), lowest_high = __reduce_min_sync(0xffffffffu, high);
    if (lane == 0) sh.common[warp] = make_int2(highest_low, lowest_high);
    if (is_active(g, slot)) {
      if (!(g.turns && slot == 1)) {
        const int in_tile = warp % 4 * 32;
        put_queries<D>(a.q, (g.q_first + token) * a.q_stride + column, a.scale_log2, g.rows - slot * kSlotRows - in_tile,
                       smem + Shape::kQ + slot * Shape::kTileBytes, in_tile, sh.unit + slot * 128 + in_tile);
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_full[slot]);
    }
    __syncwarp();
  };
  while (true) {
    wait_whole_warp(sh, &sh.segment_full[segment & 3], segment >> 2 & 1);
    if (softmax_bar_any(sh.abort_code != 0)) return;      // all eight warps meet here whatever failed, and leave together
    // A segment's q goes to shared memory before the results of the one in front leave tensor memory, so that its first scores do not have to
    // be waited for.
    const bool more = sh.segment[segment & 3].tiles > 0;
    if (more) begin(sh.segment[segment & 3]);
    if (segment > 0) {
      const Segment& g = sh.segment[(segment - 1) & 3];
      const int thread = thread_here(), warp = thread / 32, lane = thread % 32, slot = warp / 4, in_slot = thread % 128;
      const int row = row_of(g, thread), across = 2 + warp % 4;      // named barrier of the two slots' warps for the same rows
      const uint32_t t_o = sh.tmem + (static_cast<uint32_t>(warp % 4 * 32) << 16) + slot * 128 + 256;
      const bool turns = g.turns, whole = g.whole, real = row < g.rows && !(turns && slot == 1);
      if (is_active(g, slot)) {
        float4 mine = sh.end[slot][in_slot];    // m, l, n
        float f = 1.0f;
        if (turns) {                            // to the larger references of the two slots'
          const float4 its = sh.end[slot ^ 1][in_slot];
          const float m_all = fmaxf(mine.x, its.x), m_ref = finite_or_zero(m_all), n_all = fmaxf(mine.z, its.z);
          f = ex2(mine.z - finite_or_zero(n_all));
          mine = make_float4(m_all, mine.y * ex2(mine.x - m_ref) + its.y * ex2(its.x - m_ref), n_all, 0.0f);
        }
        if (whole) f *= mine.y == 0.0f || mine.z == -INFINITY ? 0.0f : ex2(mine.z - finite_or_zero(mine.x) - kProductHeadroom) / mine.y;
        float4* const its = reinterpret_cast<float4*>(smem + Shape::kHandOver) + warp % 4 * 128 + lane;      // slot 1's sums on their way to slot 0
        float4* const to = reinterpret_cast<float4*>(a.partial);       // (kept by dimension, so that a warp's 32 rows lie side by side)
        const int part = parts_of(g).slot(static_cast<int>(blockIdx.x));
        // Two neighbouring lanes write 32 bytes of one's row, then of the other's.
        int column;
        const int token = token_of(g, row, column);
        const long long place = (g.q_first + token) * a.out_stride + column, place_other = __shfl_xor_sync(0xffffffffu, place, 1);
        const bool odd = lane % 2 != 0, real_other = (row ^ 1) < g.rows;
        __nv_bfloat16* const even_row = a.out + (odd ? place_other : place) + 8 * odd;
        __nv_bfloat16* const odd_row = a.out + (odd ? place : place_other) + 8 * odd;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          uint32_t o[16];
          tmem_ld16(t_o + c, o);
          tmem_ld_wait_for(o);
#pragma unroll
          for (int b = 0; b < 16; ++b) o[b] = __float_as_uint(__uint_as_float(o[b]) * f);
          if (turns) {                          // slot 0 adds slot 1's sums to its own
            if (slot == 1) {
#pragma unroll
              for (int b = 0; b < 4; ++b)
                its[32 * b] = make_float4(__uint_as_float(o[4 * b]), __uint_as_float(o[4 * b + 1]), __uint_as_float(o[4 * b + 2]), __uint_as_float(o[4 * b + 3]));
            }
            named_bar_sync(across, 64);
            if (slot == 0) {
#pragma unroll
              for (int b = 0; b < 4; ++b) {
                const float4 x = its[32 * b];
                o[4 * b] = __float_as_uint(__uint_as_float(o[4 * b]) + x.x);
                o[4 * b + 1] = __float_as_uint(__uint_as_float(o[4 * b + 1]) + x.y);
                o[4 * b + 2] = __float_as_uint(__uint_as_float(o[4 * b + 2]) + x.z);
                o[4 * b + 3] = __float_as_uint(__uint_as_float(o[4 * b + 3]) + x.w);
              }
            }
            named_bar_sync(across, 64);
            if (slot == 1) continue;
          }
          if (whole) {
            uint32_t low[4], high[4];           // this lane's row: its first eight of sixteen dimensions, the others
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __nv_bfloat162 x = __floats2bfloat162_rn(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
              const __nv_bfloat162 y = __floats2bfloat162_rn(__uint_as_float(o[8 + 2 * e]), __uint_as_float(o[9 + 2 * e]));
              low[e] = *reinterpret_cast<const uint32_t*>(&x);
              high[e] = *reinterpret_cast<const uint32_t*>(&y);
              const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? low[e] : high[e], 1);
              if (odd) low[e] = got;            // the even row's second half
              else high[e] = got;               // the odd row's first half
            }
            if (odd ? real_other : real) *reinterpret_cast<uint4*>(even_row + c) = make_uint4(low[0], low[1], low[2], low[3]);
            if (odd ? real : real_other) *reinterpret_cast<uint4*>(odd_row + c) = make_uint4(high[0], high[1], high[2], high[3]);
          } else if (real) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              to[(static_cast<long long>(part) * (D / 4) + c / 4 + e) * kChunkRows + row] =
                  make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
          }
        }
        if (real && !whole) reinterpret_cast<float4*>(a.partial + 2ll * piece.ctas * kChunkRows * D)[static_cast<long long>(part) * kChunkRows + row] = mine;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.o_empty[slot]);
      }
      if (!whole) {
        const Parts parts = parts_of(g);
        __threadfence();
        named_bar_sync(1, kSoftmaxThreads);
        if (tid == 0) {
          const bool is_last = atomicAdd(a.tickets + parts.first, 1) == parts.last - parts.first;
          if (is_last) a.tickets[parts.first] = 0;
          s_plan.last = is_last;
        }
        named_bar_sync(1, kSoftmaxThreads);
        if (s_plan.last) {
          __threadfence();
          join_columns<D>(a, g.q_first, g.row0, g.head, g.rows, piece.ctas, parts, tid, kSoftmaxThreads);
        }
      }
      if (tid == 0) ++sh.finished;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.segment_empty[(segment - 1) & 3]);
    }
    if (!more) {
      if (tid == 0) sh.done = 1;
      return;
    }
    const Segment& g = sh.segment[segment & 3];
    const bool turns = g.turns;
    // whether the next tile is this slot's (bit 0: no), and whether that changes with each (bit 1)
    unsigned turn = turns ? 2u + slot : !is_active(g, slot);
    {
      if (turns) named_bar_sync(1, kSoftmaxThreads);       // slot 1 reads slot 0's units
      TileRows r;
      r.bounds = sh.bounds[0];
      r.offset = 0;
      const int first_row = warp % 4 * 32 + lane / 4;      // the first of this lane's four in the slot
      float ms[4], ns[4], ls[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r.unit[i] = sh.unit[(turns ? 0 : slot) * 128 + first_row + 8 * i];
        ms[i] = ns[i] = -INFINITY;
        ls[i] = 0.0f;
      }
      int settled = kBlind;
      for (int left = g.tiles; left > 0; --left) {
        const int stage = tile & 3;
        wait_whole_warp(sh, &sh.scale_full[stage], tile >> 2 & 1);
        if (!(turn & 1u)) {
          const int thread = thread_here();
          const int2 common = sh.common[thread / 32];
          const int flags = sh.flags[stage];
          r.there0 = flags & 1;
          r.there1 = flags & 2;
          r.near = flags & 4;
          r.masked = !r.there0 || !r.there1 || common.x > r.offset || common.y < r.offset + kTile - 1;
          r.scales = scales0 + stage * (2 * kTile * 4) + thread % 4 * 8;
          r.t_s = sh.tmem + (static_cast<uint32_t>(thread / 32 % 4 * 32) << 16) + thread / 128 * 128;
          const Segment& now = sh.segment[segment & 3];
          softmax_tile<D>(sh, r, thread / 128, stage, own & 1, left > now.tiles - (now.turns ? 2 : 1), settled, ms, ns, ls);
          own ^= 1u;
        }
        __syncwarp();
        if (thread_here() % 32 == 0) mbar_arrive(&sh.scale_empty[stage]);
        ++tile;
        if (thread_here() == 0) sh.tiles_done = sh.tiles_done + 1u;
        turn ^= turn >> 1 & 1u;
        r.offset += kTile;
      }
      // ---- the segment's end: from here on a thread has a row
      if (is_active(g, thread_here() / 128)) {
        const int thread = thread_here(), warp = thread / 32, lane = thread % 32, slot = warp / 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ls[i] += __shfl_xor_sync(0xffffffffu, ls[i], 1);
          ls[i] += __shfl_xor_sync(0xffffffffu, ls[i], 2);
          if (lane % 4 == 0) sh.end[slot][warp % 4 * 32 + lane / 4 + 8 * i] = make_float4(ms[i], ls[i], ns[i], 0.0f);
        }
        wait_whole_warp(sh, &sh.o_full[slot], own >> 1 & 1);
        __syncwarp();
        tc_fence_after();
        own ^= 2u;
      }
    }
    ++segment;
  }
}

template <int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
kv4_chunk_kernel(const __grid_constant__ AttentionArgs a, int* __restrict__ status, long long wait_limit) {
  using Shape = ChunkShape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ ChunkShared sh;
  __shared__ PlanShared s_plan;
  __shared__ Piece piece;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;

  pdl_wait();
  pdl_trigger();
  const ChunkPlan plan = {a.batch, a.cache.heads, a.group, a.window};
  {
    const long long total = plan.total(s_plan);
    const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
    if (static_cast<int>(blockIdx.x) >= ctas) return;
    const long long w0 = piece_start(total, ctas, blockIdx.x), w1 = piece_start(total, ctas, blockIdx.x + 1);
    if (tid == 0) piece = {total, w1, ctas, static_cast<int>(w1 - w0)};
    plan.locate(s_plan, w0);
  }

  if (tid == 0) {
    for (int i = 0; i < kScaleStages; ++i) {
      mbar_init(&sh.scale_full[i], 1);
      mbar_init(&sh.scale_empty[i], kSoftmaxWarps);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sh.k_full[i], 4);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_full[i], 4);
      mbar_init(&sh.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.q_full[i], 4);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_half[i], 4);
      mbar_init(&sh.half_done[i], 1);
      mbar_init(&sh.p_full[i], 4);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.o_empty[i], 4);
    }
    mbar_init(&sh.idle, 1);
    for (int i = 0; i < kSegmentRing; ++i) {
      mbar_init(&sh.segment_full[i], 1);
      mbar_init(&sh.segment_empty[i], kSegmentReaders);
      sh.segment[i].tiles = 0;
    }
    sh.abort_code = 0;
    sh.tiles_done = 0u;
    sh.done = 0;
    sh.finished = 0;
    fence_barrier_init();
  }
  if (warp == 12) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;                // S of slot s at columns 128 s (P over its first 64), O at 256 + 128 s
  // 512 threads at 128 registers: 256 softmax threads at 176, 128 converting ones at 88 and 128 others at 72, until the roles are done.
  if (warp < kSoftmaxWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    softmax_role<D>(a, sh, s_plan, smem, piece);
    asm volatile("setmaxnreg.dec.sync.aligned.u32 128;");
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    convert_role<D>(a, sh, smem);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (lane == 0) {
      if (warp == 12) mma_role<D>(sh, smem, tmem);
      if (warp == 13) plan_role<D>(a, plan, s_plan, sh, piece, wait_limit);
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  // (Not before every role is done: an idle warp that took its registers back at once could take those that a softmax warp is
  // still to get, and the two would wait for each other.)
  if (warp >= kSoftmaxWarps) asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
  if (sh.abort_code != 0) {
    // A role gave up: MMAs may still be on their way, which otherwise the roles have waited for.
    if (tid == 12 * 32) {
      umma_commit(&sh.idle);
      mbar_wait_landed(&sh.idle, 0);
    }
    __syncthreads();
    // What is left of the piece becomes NaN, and its units are counted, so that nobody waits for them and the next call finds the
    // counters at zero.
    ChunkCursor at;
    at.start(plan, s_plan, piece.places);
    bool unfinished = false;                  // (the last tile's time may run out when all that is left is to leave)
    for (int segment = 0; at.left > 0; ++segment) {
      const int n = at.tiles_here(), rows = at.rows(a.group);
      const bool whole = n == at.span.tiles;
      if (segment >= sh.finished) {
        unfinished = true;
        if (whole) {
          for (int x = tid; x < rows * D; x += kChunkThreads) {
            const int r = at.rt * kChunkRows + x / D;
            a.out[(at.s.first + r / a.group) * a.out_stride + (at.head * a.group + r % a.group) * D + x % D] = __float2bfloat16(__int_as_float(0x7fffffff));
          }
        } else {
          const Parts parts(piece.total, piece.ctas, piece.w1 - at.left - at.tile, at.span.tiles);
          const int slot_no = parts.slot(static_cast<int>(blockIdx.x));
          for (int x = tid; x < rows; x += kChunkThreads)
            reinterpret_cast<float4*>(a.partial + 2ll * piece.ctas * kChunkRows * D)[static_cast<long long>(slot_no) * kChunkRows + x] =
                make_float4(0.0f, __int_as_float(0x7fffffff), 0.0f, 0.0f);
          __threadfence();
          __syncthreads();
          if (tid == 0) {
            const bool is_last = atomicAdd(a.tickets + parts.first, 1) == parts.last - parts.first;
            if (is_last) a.tickets[parts.first] = 0;
            s_plan.last = is_last;
          }
          __syncthreads();
          if (s_plan.last) {
            __threadfence();
            join_columns<D>(a, at.s.first, at.rt * kChunkRows, at.head, rows, piece.ctas, parts, tid, kChunkThreads);
          }
          __syncthreads();
        }
      }
      at.advance(plan, n);
    }
    if (tid == 0 && unfinished) atomicExch(status, sh.abort_code);
  }
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

size_t kv4_chunk_partial_bytes(int head_dim, int ctas) { return 2ull * ctas * kChunkRows * (head_dim + 4) * sizeof(float); }

cudaError_t kv4_chunk_set_attributes() {
  const cudaError_t e = cudaFuncSetAttribute(kv4_chunk_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, ChunkShape<128>::kSmem);
  return e != cudaSuccess ? e : cudaFuncSetAttribute(kv4_chunk_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, ChunkShape<64>::kSmem);
}

cudaError_t launch_kv4_chunk(const AttentionArgs& a, int head_dim, int ctas, int* status, long long wait_limit, cudaStream_t st) {
  return head_dim == 128 ? launch_dependent(kv4_chunk_kernel<128>, dim3(ctas), dim3(kChunkThreads), ChunkShape<128>::kSmem, st, a, status, wait_limit)
                         : launch_dependent(kv4_chunk_kernel<64>, dim3(ctas), dim3(kChunkThreads), ChunkShape<64>::kSmem, st, a, status, wait_limit);
}

}  // namespace syfi
