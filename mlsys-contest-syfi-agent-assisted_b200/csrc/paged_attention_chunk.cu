// Attention of many rows per sequence and key head: chunks of prompts and whole prompts, on the tensor cores.
//
// A CTA (one per SM) walks its piece of the line of 128-position tiles.  A unit's up to 256 rows are two slots of 128, the M of an MMA:
//   S = Q K^T   tcgen05.mma kind::f8f6f4 straight from the cache's e4m3 bytes as TMA brings them.  A row of q, scaled by a power of two, is
//               the sum of two e4m3 terms: a bf16 value has 8 significant bits, an e4m3 term 4, so the two hold it exactly as long
//               as it is not 2^-9 of the row's largest (then to 2^-17 of that).  Both terms add into one accumulator.
//   P           softmax warps, a thread per row: the weights in f16 (2^-12 of each on average), back into tensor memory over S.
//   O += P V    kind::f16, P from tensor memory, V as f16 in shared memory.  Four warps make it from the bytes: e4m3 times the position's
//               scale relative to the unit's (a power of two that follows the largest scale met), rounded once to f16.
// The slots are out of step by half a tile: while the softmax warps of one work, the tensor core works for the other.
//
// The sum's reference follows a row's largest score only when that has grown by 2^8 (kGrowth), so O is hardly ever rescaled.
// What f16 cannot hold is computed again: a unit that meets a value scale below 2^-19 of the largest is redone row by row in f32
// (exact_row).
#include "attention_common.cuh"
#include "stream_scratch.h"

namespace syfi {

namespace {

constexpr int kTile = 128;             // positions per tile: two pages
constexpr int kChunkRows = 256;
constexpr int kChunkThreads = 512;
constexpr int kScaleStages = 4;
constexpr int kStatusChunkTimeout = 301;
constexpr int kUnitShift = 5;          // the largest value scale becomes 2^4 .. 2^5 when the unit's reference is set, ...
constexpr int kUnitGrowth = 2;         // ... and may grow to 2^7 (448 * 2^7 < 65504) before the reference follows
constexpr float kSmallestUnit = 6.103515625e-5f;   // 2^-14: f16's smallest normal number

template <int D>
struct ChunkShape {
  static constexpr int kKStages = D == 128 ? 3 : 4;
  static constexpr int kVStages = 2;
  static constexpr int kHalfStages = 2;
  static constexpr int kTileBytes = kTile * D;                    // e4m3
  static constexpr int kHalfBytes = 2 * kTileBytes;
  static constexpr int kQ = 0;                                    // [2 slots][2 terms][128 rows][D]
  static constexpr int kK = kQ + 4 * kTileBytes;
  static constexpr int kV = kK + kKStages * kTileBytes;
  static constexpr int kHalf = kV + kVStages * kTileBytes;        // [D / 64][128 positions][64] f16 per stage
  static constexpr int kScales = kHalf + kHalfStages * kHalfBytes;  // [K 128 f32][V 128 f32] per stage
  static constexpr int kRedo = kScales + kScaleStages * 2 * kTile * 4;   // [8 warps][D + 64] f32
  static constexpr int kSmem = 1024 + kRedo + 8 * (D + kKvPage) * 4;
};

// A piece of a unit, as the planning warp describes it to the others.
struct Segment {
  int tile0, tiles;                    // tiles [tile0, tile0 + tiles) of the sequence's positions
  int rows, row0;                      // rows [row0, row0 + rows) of the sequence's count * group
  int head, b, q_first;                // key head, sequence, its first row of q
  int base;                            // position of the sequence's first query
  int any_low, any_high, all_low, all_high;   // positions that any / all of the rows see
  int whole;                           // the unit lies in this piece alone
  int unit_tiles;
  long long unit_start;                // on the line
};
constexpr int kSegmentRing = 4;
constexpr int kSegmentReaders = 14;    // arrivals that free an entry: loads, MMAs, 4 converting and 8 softmax warps

struct ChunkShared {
  Segment segment[kSegmentRing];
  uint64_t segment_full[kSegmentRing], segment_empty[kSegmentRing];
  uint64_t scale_full[kScaleStages], scale_clean[kScaleStages], scale_empty[kScaleStages], k_full[4], k_empty[4], v_full[2], v_empty[2], half_full[2], half_empty[2];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2], o_empty[2], idle;
  uint32_t tmem;
  int there[kScaleStages];             // bit p: page p of the tile is there
  volatile int redo[kSegmentRing];     // of the segment: f16 did not hold a value
  volatile int abort_code;
  int finished;                        // segments of this CTA whose results are written
  int asked_k, asked_v, asked_scales;  // loads that the producer has issued
};

// The unit's reference after a tile: 2^e above every finite scale of a position that is there and seen by any row; whole warp.
// Roles that need it follow it by themselves.
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

// One row in f32 by one warp, for what the tiles cannot hold: a lane has two of a page's positions, then D / 32 dimensions.
template <int D>
__device__ __noinline__ void exact_row(const AttentionArgs& a, int base, int q_first, int b, int head, int r, float* s_q, float* s_p) {
  const int lane = threadIdx.x % 32, t = r / a.group;
  const int position = base + t, low = a.window > 0 ? max(position - a.window + 1, 0) : 0;
  const long long column = static_cast<long long>(head * a.group + r % a.group) * D;
  const __nv_bfloat16* q = a.q + (q_first + t) * a.q_stride + column;
  for (int d = lane; d < D; d += 32) s_q[d] = __bfloat162float(q[d]);
  __syncwarp();
  float m = -INFINITY, l = 0.0f, acc[D / 32] = {};
  for (int page = low / kKvPage; page * kKvPage <= position; ++page) {
    const int at = a.batch.block_table[static_cast<long long>(b) * a.batch.max_pages + page];
    if (at < 0 || at >= a.cache.num_pages) continue;
    const uint8_t* keys = kv_block<D>(a.cache, at, 0, head);
    const uint8_t* values = kv_block<D>(a.cache, at, 1, head);
    float x[2];
    for (int i = 0; i < 2; ++i) {
      const int token = lane + 32 * i, j = page * kKvPage + token;
      x[i] = -INFINITY;
      if (j >= low && j <= position) {
        float sum = 0.0f;
        for (int d = 0; d < D; d += 2) {
          const float2 f = e4m3x2_to_float2(*reinterpret_cast<const uint16_t*>(keys + token * D + d));
          sum = fmaf(s_q[d], f.x, fmaf(s_q[d + 1], f.y, sum));
        }
        x[i] = sum * *reinterpret_cast<const float*>(keys + kKvPage * D + token * 4) * a.scale_log2;
      }
    }
    float top = fmaxf(x[0], x[1]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float m_new = fmaxf(m, top), fade = ex2(m - finite_or_zero(m_new));
    l *= fade;
    for (int i = 0; i < D / 32; ++i) acc[i] *= fade;
    m = m_new;
    for (int i = 0; i < 2; ++i) {
      const float p = ex2(x[i] - finite_or_zero(m));
      l += p;
      s_p[lane + 32 * i] = p;
    }
    __syncwarp();
    const int first = max(low - page * kKvPage, 0), last = min(position - page * kKvPage, kKvPage - 1);
    for (int token = first; token <= last; ++token) {
      const float p = s_p[token] * *reinterpret_cast<const float*>(values + kKvPage * D + token * 4);
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const float2 f = e4m3x2_to_float2(*reinterpret_cast<const uint16_t*>(values + token * D + i * 64 + lane * 2));
        acc[2 * i] = fmaf(p, f.x, acc[2 * i]);
        acc[2 * i + 1] = fmaf(p, f.y, acc[2 * i + 1]);
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
    *reinterpret_cast<__nv_bfloat162*>(a.out + (q_first + t) * a.out_stride + column + i * 64 + lane * 2) =
        __floats2bfloat162_rn(acc[2 * i] * inv, acc[2 * i + 1] * inv);
}

__device__ __forceinline__ bool wait_for(ChunkShared& sh, uint64_t* bar, uint32_t parity, long long limit) {
  return mbar_wait_bounded(bar, parity, &sh.abort_code, kStatusChunkTimeout, limit);
}
__device__ __forceinline__ void wait_whole_warp(ChunkShared& sh, bool& ok, uint64_t* bar, uint32_t parity, long long limit) {
  mbar_wait_or_clear(ok, bar, parity, &sh.abort_code, kStatusChunkTimeout, limit);
}

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

// ---------------------------------------------------------------- planning (one thread)
__device__ __forceinline__ void plan_role(const AttentionArgs& a, const Plan<kTile, kChunkRows>& plan, const PlanShared& s_plan, ChunkShared& sh, int count,
                                       long long w0, long long limit) {
  Cursor<kTile, kChunkRows> at;
  at.start(plan, s_plan);
  Ring<kSegmentRing> ring;
  for (int i = 0; i < count;) {
    if (!wait_for(sh, &sh.segment_empty[ring.stage], ring.parity ^ 1u, limit)) return;
    Segment& g = sh.segment[ring.stage];
    const int rows = at.rows(a.group), base = at.s.length - at.s.count, row0 = at.rt * kChunkRows;
    const int first = base + row0 / a.group, last = base + (row0 + rows - 1) / a.group;
    g.tile0 = at.span.first + at.tile;
    g.tiles = min(at.span.tiles - at.tile, count - i);
    g.rows = rows;
    g.row0 = row0;
    g.head = at.head;
    g.b = at.b;
    g.q_first = at.s.first;
    g.base = base;
    g.any_low = a.window > 0 ? max(first - a.window + 1, 0) : 0;
    g.any_high = last;
    g.all_low = a.window > 0 ? max(last - a.window + 1, 0) : 0;
    g.all_high = first;
    g.whole = g.tiles == at.span.tiles;
    g.unit_tiles = at.span.tiles;
    g.unit_start = w0 + i - at.tile;
    mbar_arrive(&sh.segment_full[ring.stage]);
    i += g.tiles;
    ring.next();
    if (i < count) at.next_unit(plan);
  }
}

// ---------------------------------------------------------------- loads (one thread)
template <int D>
__device__ __forceinline__ void load_role(const CUtensorMap& map, const AttentionArgs& a, ChunkShared& sh, uint8_t* smem, int count, long long limit) {
  using Shape = ChunkShape<D>;
  const uint64_t keep = l2_policy_evict_normal();          // other row tiles of the sequence read the same pages
  Ring<kSegmentRing> segments;
  Ring<kScaleStages> scales;
  Ring<Shape::kKStages> keys;
  Ring<Shape::kVStages> values;
  int head = 0, next_tile = 0, left = 0, any_low = 0, any_high = 0;
  const int32_t* table = nullptr;
  int entry0 = -1, entry1 = -1;
  // table entries of the tile to ask for next: read one tile ahead
  auto entries = [&]() {
    if (left == 0) {
      if (!wait_for(sh, &sh.segment_full[segments.stage], segments.parity, limit)) return false;
      const Segment& g = sh.segment[segments.stage];
      next_tile = g.tile0;
      left = g.tiles;
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
  bool alive = entries();
  for (int i = 0; i < count && alive; ++i) {
    const int entry[2] = {entry0, entry1}, h = head;
    const bool here[2] = {entry0 >= 0 && entry0 < a.cache.num_pages, entry1 >= 0 && entry1 < a.cache.num_pages};
    const int pages = here[0] + here[1];
    if (i + 1 < count && !entries()) return;
    if (!wait_for(sh, &sh.scale_empty[scales.stage], scales.parity ^ 1u, limit)) return;
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
    if (!wait_for(sh, &sh.k_empty[keys.stage], keys.parity ^ 1u, limit)) return;
    mbar_arrive_expect_tx(&sh.k_full[keys.stage], pages * kKvPage * D);
#pragma unroll
    for (int p = 0; p < 2; ++p)
      if (here[p]) tma_load_4d(smem + Shape::kK + keys.stage * Shape::kTileBytes + p * kKvPage * D, &map, &sh.k_full[keys.stage], 0, 0, h, entry[p], keep);
    sh.asked_k = i + 1;
    keys.next();
    if (!wait_for(sh, &sh.v_empty[values.stage], values.parity ^ 1u, limit)) return;
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
__device__ __forceinline__ void mma_role(ChunkShared& sh, uint8_t* smem, uint32_t tmem, int count, long long limit) {
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
  for (int i = 0; i < count;) {
    if (!wait_for(sh, &sh.segment_full[segments.stage], segments.parity, limit)) return;
    const int n = sh.segment[segments.stage].tiles, slots = sh.segment[segments.stage].rows > 128 ? 2 : 1;
    mbar_arrive(&sh.segment_empty[segments.stage]);
    segments.next();
    for (int s = 0; s < slots; ++s)
      if (!wait_for(sh, &sh.q_full[s], segment_parity >> s & 1u, limit)) return;
    if (!wait_for(sh, &sh.k_full[keys.stage], keys.parity, limit)) return;
    tc_fence_after();
    for (int s = 0; s < slots; ++s) scores(s, keys.stage);
    umma_commit(&sh.k_empty[keys.stage]);
    keys.next();
    for (int j = 0; j < n; ++j) {
      const bool more = j + 1 < n;
      if (more && !wait_for(sh, &sh.k_full[keys.stage], keys.parity, limit)) return;
      if (!wait_for(sh, &sh.half_full[halves.stage], halves.parity, limit)) return;
#pragma unroll 1
      for (int s = 0; s < slots; ++s) {
        if (j == 0 && !wait_for(sh, &sh.o_empty[s], (segment_parity >> s & 1u) ^ 1u, limit)) return;
        if (!wait_for(sh, &sh.p_full[s], tile_parity >> s & 1u, limit)) return;
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
    i += n;
  }
}

// ---------------------------------------------------------------- values to f16, a thread per position (four warps)
template <int D>
__device__ __forceinline__ void convert_role(ChunkShared& sh, uint8_t* smem, int count, long long limit) {
  using Shape = ChunkShape<D>;
  const int t = threadIdx.x - 8 * 32, lane = threadIdx.x % 32;
  Ring<kSegmentRing> segments;
  Ring<kScaleStages> scales;
  Ring<Shape::kVStages> raw;
  Ring<Shape::kHalfStages> halves;
  bool ok = true;
  for (int i = 0; i < count;) {
    wait_whole_warp(sh, ok, &sh.segment_full[segments.stage], segments.parity, limit);
    if (!__all_sync(0xffffffffu, ok)) return;
    const Segment& g = sh.segment[segments.stage];
    const int n = g.tiles;
    int unit = -100;
    for (int j = 0; j < n; ++j) {
      float* const k_scale = reinterpret_cast<float*>(smem + Shape::kScales) + scales.stage * 2 * kTile;
      wait_whole_warp(sh, ok, &sh.scale_full[scales.stage], scales.parity, limit);
      const int there = sh.there[scales.stage], position0 = (g.tile0 + j) * kTile, any_low = g.any_low, any_high = g.any_high;
      const int e = tile_exponent(k_scale + kTile, there, position0, any_low, any_high, lane);
      if (j == 0 || e > unit + kUnitGrowth) unit = e;
      const float scale = k_scale[kTile + t];
      const bool valid = (there >> (t / kKvPage) & 1) && position0 + t >= any_low && position0 + t <= any_high;
      const bool mixed = position0 < g.all_low || position0 + kTile - 1 > g.all_high;     // some rows may see what others do not
      const float r = scale * __int_as_float((kUnitShift - unit + 127) << 23);
      // r as two f16 terms, so that the product with a byte's value is rounded once
      const __half hi = __float2half_rn(r);
      const __half2 r_hi = __half2half2(hi), r_lo = __half2half2(__float2half_rn(r - __half2float(hi)));
      wait_whole_warp(sh, ok, &sh.v_full[raw.stage], raw.parity, limit);
      const uint8_t* const from = smem + Shape::kV + raw.stage * Shape::kTileBytes;
      // Zero times NaN is NaN: where some rows see a value that is not finite and others do not, its bytes become zeros and the NaN
      // goes by way of its score to the rows that see it.
      bool bad = false;
      if (mixed && valid) {
        uint32_t over = 0u;
#pragma unroll 2
        for (int chunk = 0; chunk < D / 16; ++chunk) {
          const uint4 p = *reinterpret_cast<const uint4*>(from + swizzled<D>(t, chunk));
          over |= ((p.x & 0x7f7f7f7fu) + 0x01010101u) | ((p.y & 0x7f7f7f7fu) + 0x01010101u) | ((p.z & 0x7f7f7f7fu) + 0x01010101u) | ((p.w & 0x7f7f7f7fu) + 0x01010101u);
        }
        bad = (over & 0x80808080u) != 0u || !(fabsf(scale) <= 3.402823466e38f);
        if (bad) k_scale[t] = __int_as_float(0x7fffffff);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.scale_clean[scales.stage]);
      wait_whole_warp(sh, ok, &sh.half_empty[halves.stage], halves.parity ^ 1u, limit);
      uint8_t* const to = smem + Shape::kHalf + halves.stage * Shape::kHalfBytes + t * 128;
      if (valid && !bad) {
        uint32_t any = 0u;
#pragma unroll 2
        for (int chunk = 0; chunk < D / 16; ++chunk) {
          const uint4 p = *reinterpret_cast<const uint4*>(from + swizzled<D>(t, chunk));
          const uint32_t w[4] = {p.x, p.y, p.z, p.w};
          uint32_t h[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t bits = e4m3x2_to_half2(w[k / 2] >> (16 * (k % 2)));
            const __half2 v = *reinterpret_cast<const __half2*>(&bits);
            const __half2 y = __hfma2(v, r_hi, __hmul2(v, r_lo));
            h[k] = *reinterpret_cast<const uint32_t*>(&y);
          }
          any |= (p.x | p.y | p.z | p.w) & 0x7f7f7f7fu;
          uint8_t* const row = to + chunk / 4 * (kTile * 128);
          *reinterpret_cast<uint4*>(row + (((2 * chunk) % 8 ^ (t & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint4*>(row + (((2 * chunk + 1) % 8 ^ (t & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
        }
        if (any != 0u && fabsf(r) < kSmallestUnit) sh.redo[segments.stage] = 1;
      } else {
#pragma unroll 2
        for (int chunk = 0; chunk < D / 8; ++chunk) *reinterpret_cast<uint4*>(to + chunk / 8 * (kTile * 128) + chunk % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sh.half_full[halves.stage]);
        mbar_arrive(&sh.v_empty[raw.stage]);
        mbar_arrive(&sh.scale_empty[scales.stage]);
      }
      if (!__all_sync(0xffffffffu, ok)) return;
      scales.next();
      raw.next();
      halves.next();
    }
    if (lane == 0) mbar_arrive(&sh.segment_empty[segments.stage]);
    segments.next();
    i += n;
  }
}

// ---------------------------------------------------------------- softmax, a thread per row (eight warps, four to a slot)
// One tile: scores from tensor memory, weights back into it, the row's reference m and sum l2 (in two halves).  `fade`: what the
// unit's reference has become smaller by.
__device__ __forceinline__ void softmax_tile(uint32_t t_s, uint32_t t_o, int o_columns, const float* k_scale, bool masked, int low, int high, int there,
                                             float unit, float fade, bool first, float& m, uint64_t& l2) {
  uint32_t s[4][32];
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_ld32(t_s + 32 * c, s[c]);
  tmem_ld_wait_for(s[0]);
#pragma unroll
  for (int c = 1; c < 4; ++c) tmem_landed(s[c]);
  // times the key's scale: scores in units of the row's
#pragma unroll
  for (int c = 0; c < 4; ++c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const ulonglong2 ks = *reinterpret_cast<const ulonglong2*>(k_scale + 32 * c + 4 * e);
      float x0, x1, x2, x3;
      f32x2_unpack(f32x2_mul(f32x2_pack_bits(s[c][4 * e], s[c][4 * e + 1]), ks.x), x0, x1);
      f32x2_unpack(f32x2_mul(f32x2_pack_bits(s[c][4 * e + 2], s[c][4 * e + 3]), ks.y), x2, x3);
      s[c][4 * e] = __float_as_uint(x0);
      s[c][4 * e + 1] = __float_as_uint(x1);
      s[c][4 * e + 2] = __float_as_uint(x2);
      s[c][4 * e + 3] = __float_as_uint(x3);
    }
  }
  if (masked) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      // bit b: the tile's position 32 c + b is there and seen (low and high count from the tile's first)
      const int first_bit = low - 32 * c, last_bit = high - 32 * c;
      uint32_t bits = last_bit < 0 || first_bit > 31 || !(there >> (c / 2) & 1) ? 0u : 0xffffffffu;
      if (last_bit >= 0 && last_bit < 31) bits &= (2u << last_bit) - 1u;
      if (first_bit > 0 && first_bit <= 31) bits &= 0xffffffffu << first_bit;
#pragma unroll
      for (int b = 0; b < 32; ++b)
        if (!(bits >> b & 1u)) s[c][b] = 0xff800000u;
    }
  }
  float top4[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    top4[c] = __uint_as_float(s[c][0]);
#pragma unroll
    for (int b = 1; b < 32; ++b) top4[c] = fmaxf(top4[c], __uint_as_float(s[c][b]));
  }
  const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * unit;
  if (top > m + kGrowth) {
    const float f = ex2(m - top);       // (0 for a row that had seen nothing)
    fade *= f;
    l2 = f32x2_mul(l2, f32x2_pack(f, f));
    m = top;
  }
  if (!first && __any_sync(0xffffffffu, fade != 1.0f)) {
    for (int c = 0; c < o_columns; c += 16) {
      uint32_t o[16];
      tmem_ld16(t_o + c, o);
      tmem_ld_wait_for(o);
#pragma unroll
      for (int b = 0; b < 16; ++b) o[b] = __float_as_uint(__uint_as_float(o[b]) * fade);
      tmem_st16(t_o + c, o);
    }
  }
  const float shift = kHeadroom - finite_or_zero(m);
  const uint64_t unit2 = f32x2_pack(unit, unit), shift2 = f32x2_pack(shift, shift);
  uint64_t more = 0ull;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    uint32_t p[16];
#pragma unroll
    for (int b = 0; b < 16; ++b) {
      float x0, x1;
      f32x2_unpack(f32x2_fma(f32x2_pack_bits(s[h][2 * b], s[h][2 * b + 1]), unit2, shift2), x0, x1);
      x0 = ex2(x0);
      x1 = ex2(x1);
      uint64_t& sum = b & 1 ? more : l2;
      sum = f32x2_add(sum, f32x2_pack(x0, x1));
      p[b] = pack_half2(x0, x1);
    }
    tmem_st16(t_s + 16 * h, p);
  }
  l2 = f32x2_add(l2, more);
  tmem_st_wait();
}

// The row's part of q as two e4m3 terms of q * 2^k, its largest at 2^7 .. 2^8, into the slot's tiles; returns what a score's unit is.
template <int D>
__device__ __forceinline__ float put_query(const __nv_bfloat16* q, bool real, float scale_log2, uint8_t* hi_tile, int row) {
  uint4 raw[D / 8];
  unsigned top = 0u;
#pragma unroll
  for (int c = 0; c < D / 8; ++c) {
    raw[c] = real ? __ldg(reinterpret_cast<const uint4*>(q) + c) : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, max(w[e] & 0x7fffu, w[e] >> 16 & 0x7fffu));
  }
  const int k = top == 0u ? 0 : min(7 - (static_cast<int>(top >> 7) - 127), 120);
  const float up = copysignf(__int_as_float((k + 127) << 23), scale_log2);
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    const uint32_t w[8] = {raw[2 * c].x, raw[2 * c].y, raw[2 * c].z, raw[2 * c].w, raw[2 * c + 1].x, raw[2 * c + 1].y, raw[2 * c + 1].z, raw[2 * c + 1].w};
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x0 = __uint_as_float(w[2 * e] << 16) * up, x1 = __uint_as_float(w[2 * e] & 0xffff0000u) * up;
      const float x2 = __uint_as_float(w[2 * e + 1] << 16) * up, x3 = __uint_as_float(w[2 * e + 1] & 0xffff0000u) * up;
      const uint16_t h01 = cvt_e4m3x2(x0, x1), h23 = cvt_e4m3x2(x2, x3);
      const float2 f01 = e4m3x2_to_float2(h01), f23 = e4m3x2_to_float2(h23);
      hi[e] = h01 | static_cast<uint32_t>(h23) << 16;
      lo[e] = cvt_e4m3x2(x0 - f01.x, x1 - f01.y) | static_cast<uint32_t>(cvt_e4m3x2(x2 - f23.x, x3 - f23.y)) << 16;
    }
    const int to = swizzled<D>(row, c);
    *reinterpret_cast<uint4*>(hi_tile + to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(hi_tile + ChunkShape<D>::kTileBytes + to) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
  // (a scale of zero keeps a factor, so that -infinity stays what it is)
  return top >= 0x7f80u ? __int_as_float(0x7fffffff) : fmaxf(fabsf(scale_log2) * __int_as_float((127 - k) << 23), 1e-30f);
}

template <int D>
__device__ __forceinline__ void softmax_role(const AttentionArgs& a, ChunkShared& sh, PlanShared& s_plan, uint8_t* smem, uint32_t tmem, int count, int ctas,
                                             long long total, long long limit) {
  using Shape = ChunkShape<D>;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, slot = warp / 4;
  const uint32_t lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
  const uint32_t t_s = tmem + lanes + slot * 128, t_o = tmem + lanes + 256 + slot * 128;
  Ring<kSegmentRing> segments;
  Ring<kScaleStages> scales;
  uint32_t tile_parity = 0, segment_parity = 0;     // of this slot
  bool ok = true;
  int done = 0;                                     // segments
  for (int i = 0; i < count;) {
    wait_whole_warp(sh, ok, &sh.segment_full[segments.stage], segments.parity, limit);
    __syncwarp();
    const Segment& g = sh.segment[segments.stage];
    const int n = ok ? g.tiles : 0;
    const bool active = slot * 128 < g.rows;
    const bool real = tid < g.rows;
    float unit = 0.0f, m = -INFINITY;
    uint64_t l2 = 0ull;
    int exponent = -100;
    if (n > 0) {
      const int r = g.row0 + (real ? tid : g.rows - 1), token = r / a.group;        // (rows beyond the last copy its bounds)
      const int high = g.base + token, low = a.window > 0 ? max(high - a.window + 1, 0) : 0;
      if (active) {
        unit = put_query<D>(a.q + (g.q_first + token) * a.q_stride + (g.head * a.group + r % a.group) * D, real, a.scale_log2,
                            smem + Shape::kQ + 2 * slot * Shape::kTileBytes, tid % 128);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_full[slot]);
      }
      const int warp_low = __reduce_max_sync(0xffffffffu, low), warp_high = __reduce_min_sync(0xffffffffu, high);   // seen by every row of the warp
      for (int j = 0; j < n; ++j) {
        wait_whole_warp(sh, ok, &sh.scale_full[scales.stage], scales.parity, limit);
        wait_whole_warp(sh, ok, &sh.scale_clean[scales.stage], scales.parity, limit);
        if (active) {
          const float* const k_scale = reinterpret_cast<const float*>(smem + Shape::kScales) + scales.stage * 2 * kTile;
          const int there = sh.there[scales.stage], position0 = (g.tile0 + j) * kTile;
          const int e = tile_exponent(k_scale + kTile, there, position0, g.any_low, g.any_high, lane);
          float fade = 1.0f;
          if (j == 0) {
            exponent = e;
          } else if (e > exponent + kUnitGrowth) {
            fade = ex2(static_cast<float>(exponent - e));
            exponent = e;
          }
          wait_whole_warp(sh, ok, &sh.s_full[slot], tile_parity, limit);
          __syncwarp();
          tc_fence_after();
          softmax_tile(t_s, t_o, D, k_scale, position0 < warp_low || position0 + kTile - 1 > warp_high || there != 3, low - position0, high - position0,
                       there, unit, fade, j == 0, m, l2);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_full[slot]);
          tile_parity ^= 1u;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.scale_empty[scales.stage]);
        scales.next();
        if (!__all_sync(0xffffffffu, ok)) break;
      }
      // ---- the segment's end
      if (active) {
        wait_whole_warp(sh, ok, &sh.o_full[slot], segment_parity, limit);
        __syncwarp();
        tc_fence_after();
        segment_parity ^= 1u;
      }
    }
    if (softmax_bar_any(!ok)) return;         // all eight warps meet here whatever failed, and leave together
    const bool redo = sh.redo[segments.stage] != 0, whole = g.whole;
    if (tid == 0) sh.redo[(segments.stage + kSegmentRing - 1) % kSegmentRing] = 0;     // the segment before: everybody has read it
    const Parts parts(total, ctas, g.unit_start, g.unit_tiles);
    const int r = g.row0 + tid, token = r / a.group;
    if (active) {
      const int part = parts.slot(static_cast<int>(blockIdx.x)) * kChunkRows + tid;
      float l0, l1;
      f32x2_unpack(l2, l0, l1);
      const float l = l0 + l1, unscale = __int_as_float((exponent - kUnitShift + 127) << 23);
      const float f = whole ? (l == 0.0f ? 0.0f : unscale / l) : unscale;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(t_o + 32 * c, o);
        tmem_ld_wait_for(o);
        if (real && whole && !redo) {
          uint4* to = reinterpret_cast<uint4*>(a.out + (g.q_first + token) * a.out_stride + (g.head * a.group + r % a.group) * D + 32 * c);
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(o[8 * b + 2 * e]) * f, __uint_as_float(o[8 * b + 2 * e + 1]) * f);
              w[e] = *reinterpret_cast<const uint32_t*>(&h);
            }
            to[b] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else if (real && !whole) {
          float4* to = reinterpret_cast<float4*>(a.partial + static_cast<long long>(part) * D + 32 * c);
#pragma unroll
          for (int b = 0; b < 8; ++b)
            to[b] = make_float4(__uint_as_float(o[4 * b]) * f, __uint_as_float(o[4 * b + 1]) * f, __uint_as_float(o[4 * b + 2]) * f, __uint_as_float(o[4 * b + 3]) * f);
        }
      }
      if (real && !whole)
        reinterpret_cast<float4*>(a.partial + 2ll * ctas * kChunkRows * D)[part] = make_float4(m, l * 0.0078125f, m, redo ? 1.0f : 0.0f);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.o_empty[slot]);
    }
    bool again = whole && redo;               // whether this CTA has to redo the unit row by row
    if (!whole) {
      __threadfence();
      named_bar_sync(1, 256);
      if (tid == 0) {
        const bool is_last = atomicAdd(a.tickets + parts.first, 1) == parts.last - parts.first;
        if (is_last) a.tickets[parts.first] = 0;
        s_plan.last = is_last;
      }
      named_bar_sync(1, 256);
      if (s_plan.last) {
        __threadfence();
        const float4* stats = reinterpret_cast<const float4*>(a.partial + 2ll * ctas * kChunkRows * D);
        for (int c = parts.first; c <= parts.last; ++c) again |= __ldcg(stats + static_cast<long long>(parts.slot(c)) * kChunkRows).w != 0.0f;
        if (!again) join_parts<D, kChunkRows, 8>(a, g.q_first, g.row0, g.head, g.rows, ctas, parts, tid, 256);
      }
    }
    if (again) {
      float* const s_q = reinterpret_cast<float*>(smem + Shape::kRedo) + warp * (D + kKvPage);
      for (int x = warp; x < g.rows; x += 8) exact_row<D>(a, g.base, g.q_first, g.b, g.head, g.row0 + x, s_q, s_q + D);
    }
    if (tid == 0) sh.finished = ++done;
    i += n;
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.segment_empty[segments.stage]);
    segments.next();
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
  const Plan<kTile, kChunkRows> plan = {a.batch, a.cache.heads, a.group, a.window};
  const long long total = plan.total(s_plan);
  const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
  if (static_cast<int>(blockIdx.x) >= ctas) return;
  const long long w0 = piece_start(total, ctas, blockIdx.x), w1 = piece_start(total, ctas, blockIdx.x + 1);
  const int count = static_cast<int>(w1 - w0);
  plan.locate(s_plan, w0);

  if (tid == 0) {
    for (int i = 0; i < kScaleStages; ++i) {
      mbar_init(&sh.scale_full[i], 1);
      mbar_init(&sh.scale_clean[i], 4);         // converting warps
      mbar_init(&sh.scale_empty[i], 12);        // softmax and converting warps
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sh.k_full[i], 1);
      mbar_init(&sh.k_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.v_full[i], 1);
      mbar_init(&sh.v_empty[i], 4);
      mbar_init(&sh.half_full[i], 4);
      mbar_init(&sh.half_empty[i], 1);
      mbar_init(&sh.q_full[i], 4);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 4);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.o_empty[i], 4);
    }
    mbar_init(&sh.idle, 1);
    for (int i = 0; i < kSegmentRing; ++i) {
      mbar_init(&sh.segment_full[i], 1);
      mbar_init(&sh.segment_empty[i], kSegmentReaders);
      sh.redo[i] = 0;
    }
    sh.abort_code = 0;
    sh.finished = 0;
    sh.asked_k = sh.asked_v = sh.asked_scales = 0;
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
  // 512 threads at 128 registers are all there are: 256 of them at 56 leave 200 for each softmax thread, until the roles are done.
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    softmax_role<D>(a, sh, s_plan, smem, tmem, count, ctas, total, wait_limit);
    asm volatile("setmaxnreg.dec.sync.aligned.u32 128;");
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp < 12) {
      convert_role<D>(sh, smem, count, wait_limit);
    } else if (lane == 0) {
      if (warp == 12) mma_role<D>(sh, smem, tmem, count, wait_limit);
      if (warp == 13) load_role<D>(map, a, sh, smem, count, wait_limit);
      if (warp == 14) plan_role(a, plan, s_plan, sh, count, w0, wait_limit);
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  // (Not before every role is done: an idle warp that took its registers back at once could take those that a softmax warp is
  // still to get, and the two would wait for each other.)
  if (warp >= 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
  if (sh.abort_code != 0) {
    // A role gave up: copies and MMAs may still be on their way, which otherwise the roles have waited for.
    if (tid == 13 * 32) {
      for (int i = max(sh.asked_scales - kScaleStages, 0); i < sh.asked_scales; ++i) mbar_wait_landed(&sh.scale_full[i % kScaleStages], i / kScaleStages & 1);
      for (int i = max(sh.asked_k - Shape::kKStages, 0); i < sh.asked_k; ++i) mbar_wait_landed(&sh.k_full[i % Shape::kKStages], i / Shape::kKStages & 1);
      for (int i = max(sh.asked_v - Shape::kVStages, 0); i < sh.asked_v; ++i) mbar_wait_landed(&sh.v_full[i % Shape::kVStages], i / Shape::kVStages & 1);
    }
    if (tid == 12 * 32) {
      umma_commit(&sh.idle);
      mbar_wait_landed(&sh.idle, 0);
    }
    __syncthreads();
    // What is left of the piece becomes NaN, and its units are counted, so that nobody waits for them and the next call finds the
    // counters at zero.
    Cursor<kTile, kChunkRows> at;
    at.start(plan, s_plan);
    for (int i = 0, segment = 0; i < count; ++segment) {
      const int n = min(at.span.tiles - at.tile, count - i), rows = at.rows(a.group);
      const bool whole = n == at.span.tiles;
      const long long unit_start = w0 + i - at.tile;
      if (segment >= sh.finished) {
        if (whole) {
          for (int x = tid; x < rows * D; x += kChunkThreads) {
            const int r = at.rt * kChunkRows + x / D;
            a.out[(at.s.first + r / a.group) * a.out_stride + (at.head * a.group + r % a.group) * D + x % D] = __float2bfloat16(__int_as_float(0x7fffffff));
          }
        } else {
          const int slot_no = 2 * static_cast<int>(blockIdx.x) + (w0 >= unit_start ? 0 : 1);
          for (int x = tid; x < rows; x += kChunkThreads)
            reinterpret_cast<float4*>(a.partial + 2ll * ctas * kChunkRows * D)[static_cast<long long>(slot_no) * kChunkRows + x] =
                make_float4(0.0f, __int_as_float(0x7fffffff), 0.0f, 0.0f);
          const Parts parts(total, ctas, unit_start, at.span.tiles);
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
            join_parts<D, kChunkRows, 1>(a, at.s.first, at.rt * kChunkRows, at.head, rows, ctas, parts, tid, kChunkThreads);
          }
          __syncthreads();
        }
      }
      i += n;
      if (i < count) at.next_unit(plan);
    }
    if (tid == 0) atomicExch(status, sh.abort_code);
  }
  __syncthreads();
  if (warp == 12) {
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
