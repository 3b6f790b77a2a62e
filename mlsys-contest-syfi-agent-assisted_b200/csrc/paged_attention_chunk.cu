// Attention of many rows per sequence and key head: chunks of prompts and whole prompts, on the tensor cores.
//
// A CTA (one per SM) walks its piece of the line of 128-position tiles.  A unit's up to 256 rows are two slots of 128, the M of an MMA:
//   S = Q K^T   tcgen05.mma kind::f8f6f4 straight from the cache's e4m3 bytes as TMA brings them.  A row of q, scaled by a power of two, is
//               the sum of two e4m3 terms: a bf16 value has 8 significant bits, an e4m3 term 4, so the two hold it exactly as long
//               as it is not 2^-9 of the row's largest (then to 2^-17 of that).  Both terms add into one accumulator.
//   P           softmax warps, a lane per row and a warp per half of the tile's positions: the weights in f16 (2^-12 of each on average),
//               back into tensor memory over S.  Below 2^-21 of the row's largest they lose bits, below 2^-32 they are lost: that shows
//               only in a row whose heavier positions all have values a thousand times smaller.
//   O += P V    kind::f16, P from tensor memory, V as f16 in shared memory.  Four warps make it from the bytes: e4m3 times the position's
//               scale relative to the unit's (a power of two that follows the largest scale met), rounded once to f16.
// The slots are out of step by half a tile: while the softmax warps of one work, the tensor core works for the other.  A unit of at most
// 128 rows has them in both slots, which take turns at the tiles and add their sums up at the end; with one slot at work the chain of
// scores, weights and product, 5000 clocks for a tile, stood still in between (24 sequences of 300 .. 30000 positions, 8 rows per key head:
// 178 us, in turns 141).
//
// The sum's reference follows a row's largest score only when that has grown by 2^8 (kGrowth), so O is hardly ever rescaled.
// What f16 cannot hold is computed again: where a unit meets a value scale below 2^-19 of the largest, the rows whose sums are so small
// that its rounding could show are redone one by one in f32 (kDoubt, exact_row).  The 8192-token prompt with one such value in every key head:
// 1.4 ms instead of 0.7; all rows of the units that meet it 797 ms.
//
// What bounds it is that chain: a wide tile of 256 rows takes 5200 clocks, of which the tensor core works 2048 and the exponentials 2048
// (16 per clock).  A prompt of 8192 tokens, 32 heads of 128 over 8: 649 us (848 TFLOP/s of what is visible)
// back to back, 707 to 722 us with other memory touched in between.
#include "attention_common.cuh"
#include "stream_scratch.h"

namespace syfi {

namespace {

constexpr int kTile = 128;             // positions per tile: two pages
constexpr int kChunkRows = 256;
constexpr int kChunkThreads = 768;     // 16 softmax warps, 4 converting ones, then MMAs, loads, planning, scales
constexpr int kSoftmaxWarps = 16, kSoftmaxThreads = 512;
// What a unit costs besides its tiles, in tiles.  With 2, 3, 4, 6 (us, a flushed L2): 8192-token prompt 855, 717, 660, 674; two chunks with a window
// of 1024 141, 143, 141, 143; 8 sequences of 4 to 1000 rows 68, 68, 70, 73; a chunk of 512 behind 40000 positions 325, 324, 324, 327.
constexpr int kChunkExtra = 4;
constexpr int kSlotRows = 128;         // units of at most so many rows use one slot for their even tiles and one for their odd ones
using ChunkPlan = Plan<kTile, kChunkRows, kChunkExtra, kSlotRows>;
using ChunkCursor = Cursor<kTile, kChunkRows, kChunkExtra, kSlotRows>;
constexpr int kScaleStages = 4;
constexpr int kStatusChunkTimeout = 301;
constexpr int kNoValue = 0x7fffffff;   // in a key's scale: a NaN, and its value's bytes are not looked at
constexpr int kUnitShift = 5;          // the largest value scale becomes 2^4 .. 2^5 when the unit's reference is set, ...
constexpr int kUnitGrowth = 2;         // ... and may grow to 2^7 (448 * 2^7 < 65504) before the reference follows
constexpr float kSmallestUnit = 6.103515625e-5f;   // 2^-14: f16's smallest normal number
// A value below that is off by up to 2^-25, so a row's sum by 2^-25 of its weights' sum; where a sum is smaller than 2^-14 of it, which would
// be an error of more than 2^-11, the row is computed again.
constexpr float kDoubt = 6.103515625e-5f;

template <int D>
struct ChunkShape {
  static constexpr int kKStages = D == 128 ? 2 : 4;
  static constexpr int kVStages = D == 128 ? 3 : 4;
  static constexpr int kHalfStages = 2;
  static constexpr int kTileBytes = kTile * D;                    // e4m3
  static constexpr int kHalfBytes = 2 * kTileBytes;
  static constexpr int kQ = 0;                                    // [2 slots][2 terms][128 rows][D]
  static constexpr int kK = kQ + 4 * kTileBytes;
  static constexpr int kV = kK + kKStages * kTileBytes;
  static constexpr int kHalf = kV + kVStages * kTileBytes;        // [D / 64][128 positions][64] f16 per stage
  static constexpr int kScales = kHalf + kHalfStages * kHalfBytes;  // [K 128 f32][V 128 f32] per stage
  static constexpr int kSmem = 1024 + kScales + kScaleStages * 2 * kTile * 4;
};

// A piece of a unit, as the planning warp describes it to the others.
struct Segment {
  int tile0, tiles;                    // tiles [tile0, tile0 + tiles) of the sequence's positions; no tiles: the piece is done
  int rows, row0;                      // rows [row0, row0 + rows) of the sequence's count * group
  int head, b, q_first;                // key head, sequence, its first row of q
  int base;                            // position of the sequence's first query
  int any_low, any_high, all_low, all_high;   // positions that any / all of the rows see
  int whole;                           // the unit lies in this piece alone
  int turns;                           // rows 0 .. 127 are in both slots, which take turns at the tiles
  int first_part, last_part, first_slot;   // else: its Parts
};
__device__ __forceinline__ Parts parts_of(const Segment& g) { return {g.first_part, g.last_part, g.first_slot}; }
constexpr int kSegmentRing = 4;
constexpr int kSegmentReaders = 3 + 4 + kSoftmaxWarps;    // arrivals that free an entry: loads, MMAs, scales, converting and softmax warps

struct ChunkShared {
  Segment segment[kSegmentRing];
  uint64_t segment_full[kSegmentRing], segment_empty[kSegmentRing];
  uint64_t scale_full[kScaleStages], scale_clean[kScaleStages], scale_empty[kScaleStages], k_full[4], k_empty[4], v_full[4], v_empty[4], half_full[2], half_empty[2];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2], o_empty[2], idle;
  uint32_t tmem;
  int there[kScaleStages];             // bit p: page p of the tile is there
  int exponent[kScaleStages];          // the values' reference as of the tile: 2^exponent
  float fade[kScaleStages];            // what it has become smaller by since the slot's tile before (1: nothing)
  float top[2][2][2][128];             // [tile parity][slot][half][row]: a row's largest score in half of a tile
  float end[2][4][128];                // [slot][sum of each half, reference, values' reference][row], at a segment's end
  float unit[256];                     // of each row: what a score is worth
  volatile int redo[kSegmentRing];     // of the segment: f16 did not hold a value
  uint32_t again[kChunkRows / 32];     // bit by row: the unit's rows whose result that touched
  volatile int abort_code;
  volatile uint32_t tiles_done;        // and pages of rows that are computed again: it changes while the CTA goes on
  volatile int done;                   // every segment is
  int finished;                        // segments of this CTA whose results are written
  int asked_k, asked_v, asked_scales;  // loads that the producer has issued
};

// The unit's reference after a tile: 2^e above every finite scale of a position that is there and seen by any row; whole warp.
__device__ __forceinline__ int tile_exponent(const float* v_scale, int there, int position0, int any_low, int any_high, int lane) {
  const float4 v = reinterpret_cast<const float4*>(v_scale)[lane];
  const float x[4] = {v.x, v.y, v.z, v.w};
  unsigned top = 0u;
  const bool here = (there >> (lane / 16)) & 1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned bits = __float_as_uint(x[i]) & 0x7fffffffu;
    const int position = position0 + 4 * lane + i;
    if (here && position >= any_low && position <= any_high && bits < 0x7f800000u) top = max(top, bits);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  return max(static_cast<int>(top >> 23) - 126, -100);
}

// join_parts for partial sums that are kept by dimension: a thread has a row and sixteen of its dimensions.  Rows that have to be computed
// again (kDoubt) are noted in `again`.
template <int D>
__device__ __forceinline__ void join_columns(const AttentionArgs& a, int q_first, int unit_row0, int head, int rows, int ctas, const Parts& parts, uint32_t* again,
                                             int thread, int threads) {
  const float4* const stats = reinterpret_cast<const float4*>(a.partial + 2ll * ctas * kChunkRows * D);
  const float4* const sums = reinterpret_cast<const float4*>(a.partial);
  for (int i = thread; i < kChunkRows * (D / 16); i += threads) {
    const int row = i % kChunkRows, d16 = i / kChunkRows;
    if (row >= rows) continue;
    float m = -INFINITY, l = 0.0f, doubt = 0.0f, o[16] = {};
#pragma unroll 2
    for (int c = parts.first; c <= parts.last; ++c) {
      const long long slot = parts.slot(c);
      const float4 st = __ldcg(stats + slot * kChunkRows + row);
      float4 p[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) p[k] = __ldcg(sums + (slot * (D / 4) + 4 * d16 + k) * kChunkRows + row);
      const float m_new = fmaxf(m, st.x), m_ref = finite_or_zero(m_new), f = ex2(m - m_ref), w = ex2(st.x - m_ref);
      l = l * f + st.y * w;
      doubt = doubt * f + st.w * w;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        o[4 * k] = o[4 * k] * f + p[k].x * w;
        o[4 * k + 1] = o[4 * k + 1] * f + p[k].y * w;
        o[4 * k + 2] = o[4 * k + 2] * f + p[k].z * w;
        o[4 * k + 3] = o[4 * k + 3] * f + p[k].w * w;
      }
      m = m_new;
    }
    bool small = false;
#pragma unroll
    for (int k = 0; k < 16; ++k) small |= fabsf(o[k]) < doubt;
    if (small) atomicOr(again + row / 32, 1u << (row % 32));
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
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

// A barrier of the softmax warps that tells all of them whether any thread's `p` holds.
__device__ __forceinline__ bool softmax_bar_any(bool p) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 512, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(p))
      : "memory");
  return any != 0u;
}

// One row in f32 by one warp, for what the tiles cannot hold: a lane has two of a page's positions, then D / 32 dimensions.
template <int D>
__device__ __forceinline__ void exact_row(const AttentionArgs& a, int base, int q_first, int b, int head, int r, float* s_q, float* s_p,
                                          volatile uint32_t* going) {
  constexpr int kMine = D / 32;
  const int lane = threadIdx.x % 32, t = r / a.group;
  const int position = base + t, low = a.window > 0 ? max(position - a.window + 1, 0) : 0;
  const long long column = static_cast<long long>(head * a.group + r % a.group) * D;
  const __nv_bfloat16* q = a.q + (q_first + t) * a.q_stride + column;
  for (int d = lane; d < D; d += 32) s_q[d] = __bfloat162float(q[d]);
  __syncwarp();
  float m = -INFINITY, l = 0.0f, acc[kMine] = {};
  for (int page = low / kKvPage; page * kKvPage <= position; ++page) {
    if (lane == 0) *going = *going + 1u;       // (whatever the other warps make of it: it changes)
    const int at = a.batch.block_table[static_cast<long long>(b) * a.batch.max_pages + page];
    if (at < 0 || at >= a.cache.num_pages) continue;
    const uint8_t* keys = kv_block<D>(a.cache, at, 0, head);
    const uint8_t* values = kv_block<D>(a.cache, at, 1, head);
    float x[2];
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      const int token = lane + 32 * i, j = page * kKvPage + token;
      x[i] = -INFINITY;
      if (j >= low && j <= position) {
        float sum[2] = {};
#pragma unroll 2
        for (int c = 0; c < D; c += 16) {
          const uint4 p = *reinterpret_cast<const uint4*>(keys + token * D + c);
          const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float4 y = *reinterpret_cast<const float4*>(s_q + c + 4 * k);
            const float2 f = e4m3x2_to_float2(static_cast<uint16_t>(w[k])), g = e4m3x2_to_float2(static_cast<uint16_t>(w[k] >> 16));
            sum[0] = fmaf(y.x, f.x, fmaf(y.y, f.y, sum[0]));
            sum[1] = fmaf(y.z, g.x, fmaf(y.w, g.y, sum[1]));
          }
        }
        x[i] = (sum[0] + sum[1]) * *reinterpret_cast<const float*>(keys + kKvPage * D + token * 4) * a.scale_log2;
      }
    }
    float top = fmaxf(x[0], x[1]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float m_new = fmaxf(m, top), fade = ex2(m - finite_or_zero(m_new));
    l *= fade;
#pragma unroll
    for (int i = 0; i < kMine; ++i) acc[i] *= fade;
    m = m_new;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float p = ex2(x[i] - finite_or_zero(m));
      l += p;
      s_p[lane + 32 * i] = p;
    }
    __syncwarp();
    const int first = max(low - page * kKvPage, 0), last = min(position - page * kKvPage, kKvPage - 1);
#pragma unroll 4
    for (int token = first; token <= last; ++token) {
      const float p = s_p[token] * *reinterpret_cast<const float*>(values + kKvPage * D + token * 4);
#pragma unroll
      for (int i = 0; i < kMine; i += 2) {
        const float2 f = e4m3x2_to_float2(*reinterpret_cast<const uint16_t*>(values + token * D + lane * kMine + i));
        acc[i] = fmaf(p, f.x, acc[i]);
        acc[i + 1] = fmaf(p, f.y, acc[i + 1]);
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < kMine; i += 2)
    *reinterpret_cast<__nv_bfloat162*>(a.out + (q_first + t) * a.out_stride + column + lane * kMine + i) = __floats2bfloat162_rn(acc[i] * inv, acc[i + 1] * inv);
}

// Waits in few instructions: this kernel's roles together have more code than the instruction cache of an SM holds, and its warps spend
// much of their time in these.  So a wait only asks whether somebody gave up, and the clock is the planning thread's, which has time: it
// gives up when no tile, and no page of a row that is computed again, was finished for the limit.  (The clock in every wait: a batch of
// units of 4 to 92 rows 75.2 us instead of 68.4.  A suspend hint turned into a loop of short sleeps.)
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
      sh.abort_code = kStatusChunkTimeout;
    }
    return sh.abort_code != 0;
  }
};

__device__ __forceinline__ void plan_role(const AttentionArgs& a, const ChunkPlan& plan, const PlanShared& s_plan, ChunkShared& sh, int places,
                                          long long w1, long long total, int ctas, long long wait_limit) {
  Watch watch = {wait_limit, clock64(), 0u};
  ChunkCursor at;
  at.start(plan, s_plan, places);
  Ring<kSegmentRing> ring;
  while (true) {
    while (!mbar_try_wait(&sh.segment_empty[ring.stage], ring.parity ^ 1u))
      if (watch.over(sh)) return;
    Segment& g = sh.segment[ring.stage];
    const bool more = at.left > 0;
    const int places = more ? at.tiles_here() : 0;
    g.tiles = 0;
    if (more) {
      const int rows = at.rows(a.group), base = at.s.length - at.s.count, row0 = at.rt * kChunkRows;
      const int first = base + row0 / a.group, last = base + (row0 + rows - 1) / a.group;
      g.any_low = a.window > 0 ? max(first - a.window + 1, 0) : 0;
      g.any_high = last;
      g.tile0 = at.span.first + at.tile;
      g.tiles = places;
      if (rows <= kSlotRows) {             // places of two tiles, of which the unit's ends may want one
        const int end = min(2 * (g.tile0 + places), last / kTile + 1);
        g.tile0 = max(2 * g.tile0, g.any_low / kTile);
        g.tiles = max(end - g.tile0, 1);
      }
      g.turns = rows <= kSlotRows && g.tiles > 1;
      g.rows = rows;
      g.row0 = row0;
      g.head = at.head;
      g.b = at.b;
      g.q_first = at.s.first;
      g.base = base;
      g.all_low = a.window > 0 ? max(last - a.window + 1, 0) : 0;
      g.all_high = first;
      g.whole = places == at.span.tiles;
      const Parts parts(total, ctas, w1 - at.left - at.tile, at.span.tiles);
      g.first_part = parts.first;
      g.last_part = parts.last;
      g.first_slot = parts.first_slot;
    }
    mbar_arrive(&sh.segment_full[ring.stage]);
    if (!more) break;
    ring.next();
    at.advance(plan, places);
  }
  while (sh.done == 0 && !watch.over(sh)) __nanosleep(200);
}

// ---------------------------------------------------------------- loads (one thread)
template <int D>
__device__ __forceinline__ void load_role(const CUtensorMap& map, const AttentionArgs& a, ChunkShared& sh, uint8_t* smem) {
  using Shape = ChunkShape<D>;
  const uint64_t keep = l2_policy_evict_normal();          // other row tiles of the sequence read the same pages
  Ring<kSegmentRing> segments;
  Ring<kScaleStages> scales;
  Ring<Shape::kKStages> keys;
  Ring<Shape::kVStages> values;
  int head = 0, next_tile = 0, left = 0, any_low = 0, any_high = 0;
  const int32_t* table = nullptr;
  int entry0 = -1, entry1 = -1;
  // table entries of the tile to ask for next, read one tile ahead; false behind the last
  auto entries = [&]() {
    if (left == 0) {
      if (!wait_for(sh, &sh.segment_full[segments.stage], segments.parity)) return false;
      const Segment& g = sh.segment[segments.stage];
      next_tile = g.tile0;
      left = g.tiles;
      if (left == 0) return false;
      any_low = g.any_low;
      any_high = g.any_high;
      head = g.head;
      table = a.batch.block_table + static_cast<long long>(g.b) * a.batch.max_pages;
      mbar_arrive(&sh.segment_empty[segments.stage]);
      segments.next();
    }
    const int page = 2 * next_tile;
    entry0 = page < a.batch.max_pages && page * kKvPage <= any_high && (page + 1) * kKvPage > any_low ? __ldg(table + page) : -1;
    entry1 = page + 1 < a.batch.max_pages && (page + 1) * kKvPage <= any_high && (page + 2) * kKvPage > any_low ? __ldg(table + page + 1) : -1;
    ++next_tile;
    --left;
    return true;
  };
  // A role that gave up still arrives at barriers, which may free a stage whose copy is on its way: no copy is asked for behind that.
  auto free_stage = [&](uint64_t* bar, uint32_t parity) { return wait_for(sh, bar, parity) && sh.abort_code == 0; };
  bool more = entries();
  for (int i = 0; more; ++i) {
    const int entry[2] = {entry0, entry1}, h = head;
    const bool here[2] = {entry0 >= 0 && entry0 < a.cache.num_pages, entry1 >= 0 && entry1 < a.cache.num_pages};
    const int pages = here[0] + here[1];
    more = entries();
    if (!free_stage(&sh.scale_empty[scales.stage], scales.parity ^ 1u)) return;
    sh.there[scales.stage] = here[0] | here[1] << 1;
    mbar_arrive_expect_tx(&sh.scale_full[scales.stage], pages * 2 * kKvPage * 4);
    float* const scale = reinterpret_cast<float*>(smem + Shape::kScales) + scales.stage * 2 * kTile;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if (!here[p]) continue;
      bulk_load(scale + p * kKvPage, kv_block<D>(a.cache, entry[p], 0, h) + kKvPage * D, kKvPage * 4, &sh.scale_full[scales.stage], keep);
      bulk_load(scale + kTile + p * kKvPage, kv_block<D>(a.cache, entry[p], 1, h) + kKvPage * D, kKvPage * 4, &sh.scale_full[scales.stage], keep);
    }
    sh.asked_scales = i + 1;
    scales.next();
    if (!free_stage(&sh.k_empty[keys.stage], keys.parity ^ 1u)) return;
    mbar_arrive_expect_tx(&sh.k_full[keys.stage], pages * kKvPage * D);
#pragma unroll
    for (int p = 0; p < 2; ++p)
      if (here[p]) tma_load_4d(smem + Shape::kK + keys.stage * Shape::kTileBytes + p * kKvPage * D, &map, &sh.k_full[keys.stage], 0, 0, h, entry[p], keep);
    sh.asked_k = i + 1;
    keys.next();
    if (!free_stage(&sh.v_empty[values.stage], values.parity ^ 1u)) return;
    mbar_arrive_expect_tx(&sh.v_full[values.stage], pages * kKvPage * D);
#pragma unroll
    for (int p = 0; p < 2; ++p)
      if (here[p]) tma_load_4d(smem + Shape::kV + values.stage * Shape::kTileBytes + p * kKvPage * D, &map, &sh.v_full[values.stage], 0, 0, a.cache.heads + h, entry[p], keep);
    sh.asked_v = i + 1;
    values.next();
  }
}

// ---------------------------------------------------------------- MMAs (one thread)
template <int D>
__device__ __forceinline__ void mma_role(ChunkShared& sh, uint8_t* smem, uint32_t tmem) {
  using Shape = ChunkShape<D>;
  const uint32_t qk_desc = umma_idesc_e4m3_m128(kTile), pv_desc = umma_idesc_f16_m128_n_major(D);
  const uint64_t q_desc = D == 128 ? umma_smem_desc_sw128(smem_u32(smem + Shape::kQ)) : umma_smem_desc_sw64(smem_u32(smem + Shape::kQ));
  const uint64_t v_desc = umma_smem_desc_n_major_sw128(smem_u32(smem + Shape::kHalf), kTile * 128);
  const uint32_t q0 = static_cast<uint32_t>(q_desc), k0 = q0 + (Shape::kK - Shape::kQ) / 16, qk_hi = static_cast<uint32_t>(q_desc >> 32);
  const uint32_t v0 = static_cast<uint32_t>(v_desc), v_hi = static_cast<uint32_t>(v_desc >> 32);
  auto scores = [&](int slot, int stage) {
    const uint32_t k = k0 + stage * (Shape::kTileBytes / 16), q = q0 + slot * (2 * Shape::kTileBytes / 16), to = tmem + slot * 128;
#pragma unroll
    for (int term = 0; term < 2; ++term)
#pragma unroll
      for (int step = 0; step < D / 32; ++step)
        umma_f8_words(to, q + term * (Shape::kTileBytes / 16) + 2 * step, k + 2 * step, qk_hi, qk_desc, term + step > 0 ? 1u : 0u);
    umma_commit(&sh.s_full[slot]);
  };
  auto values = [&](int slot, int stage, uint32_t add) {
    const uint32_t v = v0 + stage * (Shape::kHalfBytes / 16), p = tmem + slot * 128;
#pragma unroll
    for (int step = 0; step < kTile / 16; ++step) umma_f16_ts_words(p + 256, p + 8 * step, v + 128 * step, v_hi, pv_desc, step == 0 ? add : 1u);
  };
  Ring<kSegmentRing> segments;
  Ring<Shape::kKStages> keys;
  Ring<Shape::kHalfStages> halves;
  uint32_t tile_parity = 0, segment_parity = 0;    // bit s: of slot s
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
        scores(j, keys.stage);
        umma_commit(&sh.k_empty[keys.stage]);
        keys.next();
      }
      for (int j = 0; j < n; ++j) {
        const int s = j & 1;
        const bool more = j + 2 < n;
        if (j < 2 && !wait_for(sh, &sh.o_empty[s], (segment_parity >> s & 1u) ^ 1u)) return;
        if (!wait_for(sh, &sh.half_full[halves.stage], halves.parity)) return;
        if (!wait_for(sh, &sh.p_full[s], tile_parity >> s & 1u)) return;
        tile_parity ^= 1u << s;
        tc_fence_after();
        values(s, halves.stage, j < 2 ? 0u : 1u);
        umma_commit(&sh.half_empty[halves.stage]);
        halves.next();
        if (more) {
          if (!wait_for(sh, &sh.k_full[keys.stage], keys.parity)) return;
          scores(s, keys.stage);
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
    for (int s = 0; s < slots; ++s) scores(s, keys.stage);
    umma_commit(&sh.k_empty[keys.stage]);
    keys.next();
    for (int j = 0; j < n; ++j) {
      const bool more = j + 1 < n;
      if (more && !wait_for(sh, &sh.k_full[keys.stage], keys.parity)) return;
      if (!wait_for(sh, &sh.half_full[halves.stage], halves.parity)) return;
#pragma unroll 1
      for (int s = 0; s < slots; ++s) {
        if (j == 0 && !wait_for(sh, &sh.o_empty[s], (segment_parity >> s & 1u) ^ 1u)) return;
        if (!wait_for(sh, &sh.p_full[s], tile_parity >> s & 1u)) return;
        tile_parity ^= 1u << s;
        tc_fence_after();
        values(s, halves.stage, j > 0 ? 1u : 0u);
        if (s + 1 == slots) umma_commit(&sh.half_empty[halves.stage]);
        if (more) scores(s, keys.stage);
        else umma_commit(&sh.o_full[s]);
      }
      halves.next();
      if (more) {
        umma_commit(&sh.k_empty[keys.stage]);
        keys.next();
      }
    }
    segment_parity ^= slots == 2 ? 3u : 1u;
  }
}

// ---------------------------------------------------------------- scales (one warp)
// Looks at a tile's scales as soon as they are there, ahead of the warps that use them.
template <int D>
__device__ __forceinline__ void scale_role(ChunkShared& sh, uint8_t* smem) {
  using Shape = ChunkShape<D>;
  const int lane = threadIdx.x % 32;
  Ring<kSegmentRing> segments;
  Ring<kScaleStages> scales;
  Ring<Shape::kVStages> values;
  int unit = -100, unit_before = -100;
  while (true) {
    wait_whole_warp(sh, &sh.segment_full[segments.stage], segments.parity);
    __syncwarp();
    const Segment& g = sh.segment[segments.stage];
    const int n = __any_sync(0xffffffffu, sh.abort_code != 0) ? 0 : g.tiles;
    if (n == 0) return;
    int position0 = g.tile0 * kTile;
    const int any_low = g.any_low, any_high = g.any_high, all_low = g.all_low, all_high = g.all_high, turns = g.turns;
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.segment_empty[segments.stage]);
    segments.next();
    for (int j = 0; j < n; ++j, position0 += kTile) {
      float* const k_scale = reinterpret_cast<float*>(smem + Shape::kScales) + scales.stage * 2 * kTile;
      wait_whole_warp(sh, &sh.scale_full[scales.stage], scales.parity);
      __syncwarp();
      const int there = sh.there[scales.stage];
      const int e = tile_exponent(k_scale + kTile, there, position0, any_low, any_high, lane);
      const int before = turns ? unit_before : unit;      // as of the tile that the same slot had last
      unit_before = unit;
      if (j == 0 || e > unit + kUnitGrowth) unit = e;
      if (lane == 0) {
        sh.exponent[scales.stage] = unit;
        sh.fade[scales.stage] = before == unit ? 1.0f : ex2(static_cast<float>(before - unit));     // (nothing uses a slot's first)
      }
      // (in every tile: a wait by parity is one for this use of the stage only where the use before it is known to be over)
      wait_whole_warp(sh, &sh.v_full[values.stage], values.parity);
      if (position0 < all_low || position0 + kTile - 1 > all_high) {
        // Some rows may see what others do not, and zero times NaN is NaN: the bytes of a value that is not finite are taken for zeros, and
        // the NaN goes by way of its score to the rows that see it.
        const uint8_t* const from = smem + Shape::kV + values.stage * Shape::kTileBytes;
#pragma unroll 1
        for (int t = lane; t < kTile; t += 32) {
          if (!(there >> (t / kKvPage) & 1) || position0 + t < any_low || position0 + t > any_high) continue;
          uint32_t over = 0u;
#pragma unroll
          for (int chunk = 0; chunk < D / 16; ++chunk) {
            const uint4 p = *reinterpret_cast<const uint4*>(from + swizzled<D>(t, chunk));
            over |= ((p.x & 0x7f7f7f7fu) + 0x01010101u) | ((p.y & 0x7f7f7f7fu) + 0x01010101u) | ((p.z & 0x7f7f7f7fu) + 0x01010101u) | ((p.w & 0x7f7f7f7fu) + 0x01010101u);
          }
          if ((over & 0x80808080u) != 0u || !(fabsf(k_scale[kTile + t]) <= 3.402823466e38f)) k_scale[t] = __int_as_float(kNoValue);
        }
        fence_proxy_async_smem();              // in front of the copy that fills these scales next
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.scale_clean[scales.stage]);
      scales.next();
      values.next();
    }
  }
}

// ---------------------------------------------------------------- values to f16, a thread per position (four warps)
template <int D>
__device__ __forceinline__ void convert_role(ChunkShared& sh, uint8_t* smem) {
  using Shape = ChunkShape<D>;
  const int t = threadIdx.x - kSoftmaxThreads, lane = threadIdx.x % 32;
  Ring<kSegmentRing> segments;
  Ring<kScaleStages> scales;
  Ring<Shape::kVStages> raw;
  Ring<Shape::kHalfStages> halves;
  while (true) {
    wait_whole_warp(sh, &sh.segment_full[segments.stage], segments.parity);
    __syncwarp();
    const Segment& g = sh.segment[segments.stage];
    const int n = __any_sync(0xffffffffu, sh.abort_code != 0) ? 0 : g.tiles;
    if (n == 0) return;
    int position = g.tile0 * kTile + t;
    const int any_low = g.any_low, any_high = g.any_high;
    for (int j = 0; j < n; ++j, position += kTile) {
      const float* const k_scale = reinterpret_cast<const float*>(smem + Shape::kScales) + scales.stage * 2 * kTile;
      wait_whole_warp(sh, &sh.scale_clean[scales.stage], scales.parity);
      // what to multiply with; where there is no such value, zeros
      const float scale = k_scale[kTile + t] * __int_as_float((kUnitShift - sh.exponent[scales.stage] + 127) << 23);
      const bool valid = (sh.there[scales.stage] >> (t / kKvPage) & 1) && position >= any_low && position <= any_high && __float_as_int(k_scale[t]) != kNoValue;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.scale_empty[scales.stage]);
      scales.next();
      wait_whole_warp(sh, &sh.v_full[raw.stage], raw.parity);
      wait_whole_warp(sh, &sh.half_empty[halves.stage], halves.parity ^ 1u);
      __syncwarp();
      const uint8_t* const from = smem + Shape::kV + raw.stage * Shape::kTileBytes;
      uint8_t* const to = smem + Shape::kHalf + halves.stage * Shape::kHalfBytes + t * 128;
      if (valid) {
        // the factor as two f16 terms, so that the product with a byte's value is rounded once
        const __half hi = __float2half_rn(scale);
        const __half2 r_hi = __half2half2(hi), r_lo = __half2half2(__float2half_rn(scale - __half2float(hi)));
        uint32_t any = 0u;
#pragma unroll 1
        for (int part = 0; part < D / 64; ++part) {
          uint4 p[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) p[c] = *reinterpret_cast<const uint4*>(from + swizzled<D>(t, 4 * part + c));
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t w[4] = {p[c].x, p[c].y, p[c].z, p[c].w};
            any |= w[0] | w[1] | w[2] | w[3];
            uint32_t h[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t bits = e4m3x2_to_half2(w[k / 2] >> (16 * (k % 2)));
              const __half2 v = *reinterpret_cast<const __half2*>(&bits);
              const __half2 y = __hfma2(v, r_hi, __hmul2(v, r_lo));
              h[k] = *reinterpret_cast<const uint32_t*>(&y);
            }
            uint8_t* const row = to + part * (kTile * 128);
            *reinterpret_cast<uint4*>(row + ((2 * c ^ (t & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(row + ((2 * c + 1 ^ (t & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
          }
        }
        if (fabsf(scale) < kSmallestUnit && (any & 0x7f7f7f7fu) != 0u) sh.redo[segments.stage] = 1;
      } else {
#pragma unroll 1
        for (int chunk = 0; chunk < D / 8; ++chunk) *reinterpret_cast<uint4*>(to + chunk / 8 * (kTile * 128) + chunk % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sh.half_full[halves.stage]);
        mbar_arrive(&sh.v_empty[raw.stage]);
        if (j + 1 == n) mbar_arrive(&sh.segment_empty[segments.stage]);
      }
      if (__any_sync(0xffffffffu, sh.abort_code != 0)) return;
      raw.next();
      halves.next();
    }
    segments.next();
  }
}

// ---------------------------------------------------------------- softmax, a lane per row and half of a tile (sixteen warps, eight to a slot)
__device__ __forceinline__ ulonglong2 ld_shared_pairs(uint32_t at) {
  ulonglong2 v;
  asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(v.x), "=l"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float ld_shared_f32(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared_f32(uint32_t at, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }

// One half of a tile's row: 64 scores from tensor memory, their weights back into it, the row's reference m and this half's sum l.  The
// partner warp has the other 64; the two agree on the row's largest score through shared memory (`top`: this warp's places, `other`: the
// partner's), and only behind that barrier, when both have read their scores, write weights over them.  unit_at, fade_at: where the row's
// unit and what the values' reference has become smaller by lie.  low, high: what the row sees, counted from the first of the 64.
template <int D>
__device__ __forceinline__ void softmax_half(uint32_t t_s, uint32_t t_o, int half, uint32_t k_scale, bool masked, int low, int high, bool there,
                                             uint32_t unit_at, uint32_t fade_at, bool first, uint32_t top, uint32_t other, int barrier, float& m, float& l) {
  uint32_t s[2][32];
  tmem_ld32(t_s + half * 64, s[0]);
  tmem_ld32(t_s + half * 64 + 32, s[1]);
  tmem_ld_wait_for(s[0]);
  tmem_landed(s[1]);
  // times the keys' scales: in units of the row's
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const ulonglong2 ks = ld_shared_pairs(k_scale + 4 * (32 * c + 4 * e));
      float x0, x1, x2, x3;
      f32x2_unpack(f32x2_mul(f32x2_pack_bits(s[c][4 * e], s[c][4 * e + 1]), ks.x), x0, x1);
      f32x2_unpack(f32x2_mul(f32x2_pack_bits(s[c][4 * e + 2], s[c][4 * e + 3]), ks.y), x2, x3);
      s[c][4 * e] = __float_as_uint(x0);
      s[c][4 * e + 1] = __float_as_uint(x1);
      s[c][4 * e + 2] = __float_as_uint(x2);
      s[c][4 * e + 3] = __float_as_uint(x3);
    }
  }
  if (__builtin_expect(masked, 0)) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int first_bit = low - 32 * c, last_bit = high - 32 * c;
      uint32_t bits = last_bit < 0 || first_bit > 31 || !there ? 0u : 0xffffffffu;
      if (last_bit >= 0 && last_bit < 31) bits &= (2u << last_bit) - 1u;
      if (first_bit > 0 && first_bit <= 31) bits &= 0xffffffffu << first_bit;
#pragma unroll
      for (int b = 0; b < 32; ++b)
        if (!(bits >> b & 1u)) s[c][b] = 0xff800000u;
    }
  }
  float t0 = __uint_as_float(s[0][0]), t1 = __uint_as_float(s[1][0]);
#pragma unroll
  for (int b = 1; b < 32; ++b) {
    t0 = fmaxf(t0, __uint_as_float(s[0][b]));
    t1 = fmaxf(t1, __uint_as_float(s[1][b]));
  }
  t0 = fmaxf(t0, t1);
  st_shared_f32(top, t0);
  named_bar_sync(barrier, 64);
  const float unit = ld_shared_f32(unit_at);
  float fade = ld_shared_f32(fade_at);
  t0 = fmaxf(t0, ld_shared_f32(other)) * unit;
  if (t0 > m + kGrowth) {
    const float f = ex2(m - t0);       // (0 for a row that had seen nothing)
    fade *= f;
    l *= f;
    m = t0;
  }
  if (!first && __any_sync(0xffffffffu, fade != 1.0f)) {      // (the partner comes to the same, and has the other dimensions)
#pragma unroll 1
    for (int c = 0; c < D / 2; c += 8) {
      uint32_t o[8];
      tmem_ld8(t_o + c, o);
      tmem_ld_wait_for(o);
#pragma unroll
      for (int b = 0; b < 8; ++b) o[b] = __float_as_uint(__uint_as_float(o[b]) * fade);
      tmem_st8(t_o + c, o);
    }
  }
  const float shift = kHeadroom - finite_or_zero(m);
  const uint64_t unit2 = f32x2_pack(unit, unit), shift2 = f32x2_pack(shift, shift);
  float more = 0.0f;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    uint32_t p[8];
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const int at = 16 * (h % 2) + 2 * b;
      float x0, x1;
      f32x2_unpack(f32x2_fma(f32x2_pack_bits(s[h / 2][at], s[h / 2][at + 1]), unit2, shift2), x0, x1);
      x0 = ex2(x0);
      x1 = ex2(x1);
      l += x0;
      more += x1;
      p[b] = pack_half2(x0, x1);
    }
    tmem_st8(t_s + half * 32 + 8 * h, p);
  }
  l += more;
  tmem_st_wait();
}

// Sixteen rows of q (rows0 and on of the warp's 32) as two e4m3 terms of q * 2^k each, the row's largest at 2^7 .. 2^8, into the slot's
// tiles (row0: the warp's first row in the tile; rows: how many it has; mine: where this lane's row begins in q).  D / 8 lanes read a row,
// all under way together.  units: what a score of each row is worth.
template <int D>
__device__ __forceinline__ void put_queries(const __nv_bfloat16* q, long long mine, float scale_log2, int rows0, int rows, uint8_t* hi_tile, int row0, float* units) {
  constexpr int kLanes = D / 8, kTogether = 32 / kLanes, kBatch = 16 / kTogether;      // rows at a time
  const int lane = threadIdx.x % 32, part = lane % kLanes;
  {
    const int at = rows0;
    uint4 raw[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int row = at + b * kTogether + lane / kLanes;
      const long long from = __shfl_sync(0xffffffffu, mine, row);
      raw[b] = make_uint4(0u, 0u, 0u, 0u);
      if (row < rows) raw[b] = __ldg(reinterpret_cast<const uint4*>(q + from) + part);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int row = at + b * kTogether + lane / kLanes;
      const uint32_t w[4] = {raw[b].x, raw[b].y, raw[b].z, raw[b].w};
      unsigned top = 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, max(w[e] & 0x7fffu, w[e] >> 16 & 0x7fffu));
#pragma unroll
      for (int d = kLanes / 2; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
      const int k = top == 0u ? 0 : min(7 - (static_cast<int>(top >> 7) - 127), 120);
      const float up = copysignf(__int_as_float((k + 127) << 23), scale_log2);
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x0 = __uint_as_float(w[2 * e] << 16) * up, x1 = __uint_as_float(w[2 * e] & 0xffff0000u) * up;
        const float x2 = __uint_as_float(w[2 * e + 1] << 16) * up, x3 = __uint_as_float(w[2 * e + 1] & 0xffff0000u) * up;
        const uint16_t h01 = cvt_e4m3x2(x0, x1), h23 = cvt_e4m3x2(x2, x3);
        const float2 f01 = e4m3x2_to_float2(h01), f23 = e4m3x2_to_float2(h23);
        hi[e] = h01 | static_cast<uint32_t>(h23) << 16;
        lo[e] = cvt_e4m3x2(x0 - f01.x, x1 - f01.y) | static_cast<uint32_t>(cvt_e4m3x2(x2 - f23.x, x3 - f23.y)) << 16;
      }
      // (a row that is not finite is NaN throughout, so that the mask takes its scores out like any other's)
      if (top >= 0x7f80u) hi[0] = hi[1] = lo[0] = lo[1] = 0x7f7f7f7fu;
      uint8_t* const to = hi_tile + swizzled<D>(row0 + row, part / 2) + part % 2 * 8;
      *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
      *reinterpret_cast<uint2*>(to + ChunkShape<D>::kTileBytes) = make_uint2(lo[0], lo[1]);
      // (a scale of zero keeps a factor, f32's smallest normal number, so that -infinity stays what it is)
      if (part == 0) units[row] = fmaxf(fabsf(scale_log2) * __int_as_float((127 - k) << 23), 1.17549435e-38f);
    }
  }
}

template <int D>
__device__ __forceinline__ void softmax_role(const AttentionArgs& a, ChunkShared& sh, PlanShared& s_plan, uint8_t* smem, uint32_t tmem, int ctas) {
  using Shape = ChunkShape<D>;
  // warps 0-7: slot 0, 8-15: slot 1; of each, the first four have a tile's first 64 positions and the first half of the dimensions
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, slot = warp / 8, half = warp / 4 % 2, in_slot = warp % 4 * 32 + lane;
  const int pair = 2 + slot * 4 + warp % 4;        // named barrier of the two warps of a row
  const int across = 2 + half * 4 + warp % 4;      // between tiles: of the two slots' warps, for the same rows and dimensions
  const uint32_t lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
  const uint32_t t_s = tmem + lanes + slot * 128, t_o = t_s + 256 + half * (D / 2), scales0 = smem_u32(smem) + Shape::kScales + half * 256;
  static_assert(kSegmentRing == 4 && kScaleStages == 4, "stage and parity are bits of a counter");
  uint32_t segment = 0, tile = 0, own = 0, own_segments = 0;       // segments and tiles so far, and those of this slot
  int exponent = 0;
  while (true) {
    wait_whole_warp(sh, &sh.segment_full[segment & 3], segment >> 2 & 1);
    if (softmax_bar_any(sh.abort_code != 0)) return;      // all sixteen warps meet here whatever failed, and leave together
    if (tid < kChunkRows / 32) sh.again[tid] = 0u;        // (the segment before is over, and what this one notes comes behind the next such barrier)
    const Segment& g = sh.segment[segment & 3];
    if (g.tiles == 0) {
      if (tid == 0) sh.done = 1;
      return;
    }
    // whether the next tile is this slot's (bit 0: no), and whether that changes with each (bit 1)
    unsigned turn = g.turns ? 2u + slot : g.rows <= slot * kSlotRows;
    float m = -INFINITY, l = 0.0f;
    int token_of_row = 0, column_of_row = 0;         // of this thread's row, in q and out
    {
      int low, high;
      {
        const int r = g.row0 + min((g.turns ? 0 : slot * kSlotRows) + in_slot, g.rows - 1), token = r / a.group;        // (rows beyond the last copy its bounds)
        token_of_row = g.q_first + token;
        column_of_row = (g.head * a.group + r - token * a.group) * D;
        high = g.base + token;
        low = a.window > 0 ? max(high - a.window + 1, 0) : 0;
      }
      if (turn != 1u) {
        const int in_tile = warp % 4 * 32;
        put_queries<D>(a.q, token_of_row * a.q_stride + column_of_row, a.scale_log2, half * 16, g.rows - (g.turns ? 0 : slot * kSlotRows) - in_tile,
                       smem + Shape::kQ + 2 * slot * Shape::kTileBytes, in_tile, sh.unit + slot * 128 + in_tile);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_full[slot]);
        named_bar_sync(pair, 64);
      }
      // from here on positions count from the first of this warp's half of the segment's first tile
      const int position0 = g.tile0 * kTile + half * 64;
      low -= position0;
      high -= position0;
      bool first = true;
      for (int left = g.tiles; left > 0; --left) {
        const int stage = tile & 3;
        wait_whole_warp(sh, &sh.scale_clean[stage], tile >> 2 & 1);
        if (!(turn & 1u)) {
          wait_whole_warp(sh, &sh.s_full[slot], own & 1);
          __syncwarp();
          tc_fence_after();
          const bool there = sh.there[stage] >> half & 1;
          const uint32_t top = smem_u32(&sh.top[own & 1][slot][0][in_slot]);
          softmax_half<D>(t_s, t_o, half, scales0 + stage * (2 * kTile * 4), !there || __any_sync(0xffffffffu, low > 0 || high < 63), low, high, there,
                          smem_u32(&sh.unit[slot * 128 + in_slot]), smem_u32(&sh.fade[stage]), first, top + half * 512, top + (half ^ 1) * 512, pair, m, l);
          tc_fence_before();
          exponent = sh.exponent[stage];
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_full[slot]);
          ++own;
          first = false;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.scale_empty[stage]);
        ++tile;
        if (tid == 0) sh.tiles_done = sh.tiles_done + 1u;
        turn ^= turn >> 1 & 1u;
        low -= kTile;
        high -= kTile;
        // (a warp that failed keeps its partner company at their barrier until the segment's end)
      }
      // ---- the segment's end
      if (turn != 1u) {
        wait_whole_warp(sh, &sh.o_full[slot], own_segments & 1);
        __syncwarp();
        tc_fence_after();
        ++own_segments;
        sh.end[slot][half][in_slot] = l;
        if (half == 0) {
          sh.end[slot][2][in_slot] = m;
          sh.end[slot][3][in_slot] = __int_as_float((exponent - kUnitShift + 127) << 23);
        }
      }
    }
    if (softmax_bar_any(sh.abort_code != 0)) return;
    const bool turns = g.turns, active = turn != 1u, redo = sh.redo[segment & 3] != 0, whole = g.whole;
    const int row = (turns ? 0 : slot * kSlotRows) + in_slot;
    const bool real = row < g.rows && !(turns && slot == 1);
    if (tid == 0) sh.redo[(segment + 3) & 3] = 0;     // the segment before: everybody has read it
    if (active) {
      l = sh.end[slot][0][in_slot] + sh.end[slot][1][in_slot];
      float f = __int_as_float((exponent - kUnitShift + 127) << 23), doubt = redo ? kDoubt * l * f : 0.0f;
      if (turns) {                            // to the larger reference of the two slots'
        const float(&its)[4][128] = sh.end[slot ^ 1];
        const float its_m = its[2][in_slot], all = fmaxf(m, its_m), ref = finite_or_zero(all), fade = ex2(m - ref), its_l = (its[0][in_slot] + its[1][in_slot]) * ex2(its_m - ref);
        l = l * fade + its_l;
        doubt = redo ? doubt * fade + kDoubt * its_l * its[3][in_slot] : 0.0f;
        m = all;
        f *= fade;
      }
      if (whole) {
        const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
        f = l == 0.0f ? 0.0f : f / l;
        doubt *= inverse;
      }
      bool small = false;
      // Rows leave through the slot's q tiles, which nothing reads any more: 32 rows of D bytes per warp (half of the dimensions), swizzled,
      // then D / 16 lanes write a row's half.  Partial sums are kept by dimension, so that a warp's 32 rows lie side by side.
      uint8_t* const stage = smem + Shape::kQ + 2 * slot * Shape::kTileBytes + (half * 4 + warp % 4) * (32 * D);
      float4* const to = reinterpret_cast<float4*>(a.partial);
      float4* const its = reinterpret_cast<float4*>(smem + Shape::kQ + 2 * Shape::kTileBytes + (half * 4 + warp % 4) * (32 * D)) + lane;   // of slot 1's q tiles
      const int part = parts_of(g).slot(static_cast<int>(blockIdx.x));
#pragma unroll 1
      for (int c = 0; c < D / 16; c += 2) {
        uint32_t o[16];
        tmem_ld16(t_o + 8 * c, o);
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
        if (redo) {
#pragma unroll
          for (int b = 0; b < 16; ++b) small |= fabsf(__uint_as_float(o[b])) < doubt;
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if (whole) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(o[8 * b + 2 * e]), __uint_as_float(o[8 * b + 2 * e + 1]));
              w[e] = *reinterpret_cast<const uint32_t*>(&h);
            }
            *reinterpret_cast<uint4*>(stage + lane * D + ((D == 128 ? (c + b) ^ (lane & 7) : (c + b) ^ (lane >> 1 & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          } else if (real) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
              to[(static_cast<long long>(part) * (D / 4) + half * (D / 8) + 2 * (c + b) + e) * kChunkRows + row] =
                  make_float4(__uint_as_float(o[8 * b + 4 * e]), __uint_as_float(o[8 * b + 4 * e + 1]), __uint_as_float(o[8 * b + 4 * e + 2]),
                              __uint_as_float(o[8 * b + 4 * e + 3]));
          }
        }
      }
      if (whole && real && small) atomicOr(&sh.again[row / 32], 1u << (row % 32));
      if (whole && !(turns && slot == 1)) {
        __syncwarp();
        constexpr int kLanes = D / 16, kTogether = 32 / kLanes;
        const long long mine = token_of_row * a.out_stride + column_of_row + half * (D / 2);
#pragma unroll 4
        for (int at = 0; at < 32; at += kTogether) {
          const int line = at + lane / kLanes;
          const long long begin = __shfl_sync(0xffffffffu, mine, line);
          const uint4 p = *reinterpret_cast<const uint4*>(stage + line * D + ((D == 128 ? (lane % kLanes) ^ (line & 7) : (lane % kLanes) ^ (line >> 1 & 3)) << 4));
          if (slot * 128 + warp % 4 * 32 + line < g.rows) *(reinterpret_cast<uint4*>(a.out + begin) + lane % kLanes) = p;
        }
      }
      if (real && !whole && half == 0)
        reinterpret_cast<float4*>(a.partial + 2ll * ctas * kChunkRows * D)[static_cast<long long>(part) * kChunkRows + row] = make_float4(m, l, 0.0f, doubt);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.o_empty[slot]);
    }
    bool again = whole && redo;               // whether this CTA has to look for rows to compute again
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
        join_columns<D>(a, g.q_first, g.row0, g.head, g.rows, ctas, parts, sh.again, tid, kSoftmaxThreads);
        again = true;
      }
    }
    if (again) {
      named_bar_sync(1, kSoftmaxThreads);     // all rows are written, all notes made
      float* const s_q = reinterpret_cast<float*>(smem + Shape::kQ) + warp * (D + kKvPage);      // (nothing reads the q tiles any more)
      const bool any = __any_sync(0xffffffffu, lane < kChunkRows / 32 && sh.again[lane] != 0u);
      for (int x = warp; any && x < g.rows; x += kSoftmaxWarps)
        if (sh.again[x / 32] >> (x % 32) & 1u) exact_row<D>(a, g.base, g.q_first, g.b, g.head, g.row0 + x, s_q, s_q + D, &sh.tiles_done);
    }
    if (tid == 0) ++sh.finished;
    // (the q tiles are written again behind this: by this warp's rows' own stage only when both warps of a row are through)
    if (active) named_bar_sync(10 + slot, 256);
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.segment_empty[segment & 3]);
    ++segment;
  }
}

template <int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
attention_chunk_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ AttentionArgs a, int* __restrict__ status,
                       long long wait_limit) {
  using Shape = ChunkShape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ ChunkShared sh;
  __shared__ PlanShared s_plan;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;

  pdl_wait();
  pdl_trigger();
  const ChunkPlan plan = {a.batch, a.cache.heads, a.group, a.window};
  const long long total = plan.total(s_plan);
  const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
  if (static_cast<int>(blockIdx.x) >= ctas) return;
  const long long w0 = piece_start(total, ctas, blockIdx.x), w1 = piece_start(total, ctas, blockIdx.x + 1);
  const int places = static_cast<int>(w1 - w0);
  plan.locate(s_plan, w0);

  if (tid == 0) {
    for (int i = 0; i < kScaleStages; ++i) {
      mbar_init(&sh.scale_full[i], 1);
      mbar_init(&sh.scale_clean[i], 1);
      mbar_init(&sh.scale_empty[i], kSoftmaxWarps + 4);   // softmax and converting warps
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sh.k_full[i], 1);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_full[i], 1);
      mbar_init(&sh.v_empty[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.half_full[i], 4);
      mbar_init(&sh.half_empty[i], 1);
      mbar_init(&sh.q_full[i], 8);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 8);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.o_empty[i], 8);
    }
    mbar_init(&sh.idle, 1);
    for (int i = 0; i < kSegmentRing; ++i) {
      mbar_init(&sh.segment_full[i], 1);
      mbar_init(&sh.segment_empty[i], kSegmentReaders);
      sh.redo[i] = 0;
    }
    sh.abort_code = 0;
    sh.tiles_done = 0u;
    sh.done = 0;
    sh.finished = 0;
    sh.asked_k = sh.asked_v = sh.asked_scales = 0;
    fence_barrier_init();
  }
  if (warp == 20) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;                // S of slot s at columns 128 s (P over its first 64), O at 256 + 128 s
  // 768 threads at 80 registers: 256 of them at 48 leave 96 for each softmax thread, until the roles are done.
  if (warp < kSoftmaxWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
    softmax_role<D>(a, sh, s_plan, smem, tmem, ctas);
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp < 20) {
      convert_role<D>(sh, smem);
    } else if (warp == 23) {
      scale_role<D>(sh, smem);
    } else if (lane == 0) {
      if (warp == 20) mma_role<D>(sh, smem, tmem);
      if (warp == 21) load_role<D>(map, a, sh, smem);
      if (warp == 22) plan_role(a, plan, s_plan, sh, places, w1, total, ctas, wait_limit);
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  // (Not before every role is done: an idle warp that took its registers back at once could take those that a softmax warp is
  // still to get, and the two would wait for each other.)
  if (warp >= kSoftmaxWarps) asm volatile("setmaxnreg.inc.sync.aligned.u32 80;");
  if (sh.abort_code != 0) {
    // A role gave up: copies and MMAs may still be on their way, which otherwise the roles have waited for.
    if (tid == 21 * 32) {
      for (int i = max(sh.asked_scales - kScaleStages, 0); i < sh.asked_scales; ++i) mbar_wait_landed(&sh.scale_full[i % kScaleStages], i / kScaleStages & 1);
      for (int i = max(sh.asked_k - Shape::kKStages, 0); i < sh.asked_k; ++i) mbar_wait_landed(&sh.k_full[i % Shape::kKStages], i / Shape::kKStages & 1);
      for (int i = max(sh.asked_v - Shape::kVStages, 0); i < sh.asked_v; ++i) mbar_wait_landed(&sh.v_full[i % Shape::kVStages], i / Shape::kVStages & 1);
    }
    if (tid == 20 * 32) {
      umma_commit(&sh.idle);
      mbar_wait_landed(&sh.idle, 0);
    }
    __syncthreads();
    // What is left of the piece becomes NaN, and its units are counted, so that nobody waits for them and the next call finds the
    // counters at zero.
    ChunkCursor at;
    at.start(plan, s_plan, places);
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
          const Parts parts(total, ctas, w1 - at.left - at.tile, at.span.tiles);
          const int slot_no = parts.slot(static_cast<int>(blockIdx.x));
          for (int x = tid; x < rows; x += kChunkThreads)
            reinterpret_cast<float4*>(a.partial + 2ll * ctas * kChunkRows * D)[static_cast<long long>(slot_no) * kChunkRows + x] =
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
            join_columns<D>(a, at.s.first, at.rt * kChunkRows, at.head, rows, ctas, parts, sh.again, tid, kChunkThreads);
          }
          __syncthreads();
        }
      }
      at.advance(plan, n);
    }
    if (tid == 0 && unfinished) atomicExch(status, sh.abort_code);
  }
  __syncthreads();
  if (warp == 20) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The cache as [pages][kinds * heads][rows of D bytes][D], boxes of a block's 64 token rows.
bool cache_map(CUtensorMap* m, const KvCache& c, int head_dim) {
  const EncodeTiledFn fn = driver().encode_tiled;
  if (!fn) return false;
  const cuuint64_t block = static_cast<cuuint64_t>(kKvPage) * (head_dim + 4);
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim), block / head_dim, static_cast<cuuint64_t>(c.kinds) * c.heads, static_cast<cuuint64_t>(c.num_pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(head_dim), block, static_cast<cuuint64_t>(c.page_stride)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(head_dim), kKvPage, 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, c.base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

size_t chunk_partial_bytes(int head_dim, int ctas) { return 2ull * ctas * kChunkRows * (head_dim + 4) * sizeof(float); }

cudaError_t chunk_set_attributes() {
  const cudaError_t e = cudaFuncSetAttribute(attention_chunk_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, ChunkShape<128>::kSmem);
  return e != cudaSuccess ? e : cudaFuncSetAttribute(attention_chunk_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, ChunkShape<64>::kSmem);
}

cudaError_t launch_chunk(const AttentionArgs& a, int head_dim, int ctas, int* status, long long wait_limit, cudaStream_t st) {
  CUtensorMap map;
  if (!cache_map(&map, a.cache, head_dim)) return cudaErrorInvalidValue;
  return head_dim == 128 ? launch_dependent(attention_chunk_kernel<128>, dim3(ctas), dim3(kChunkThreads), ChunkShape<128>::kSmem, st, map, a, status, wait_limit)
                         : launch_dependent(attention_chunk_kernel<64>, dim3(ctas), dim3(kChunkThreads), ChunkShape<64>::kSmem, st, map, a, status, wait_limit);
}

}  // namespace syfi
