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
constexpr int kFlagRing = 4;
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

struct ChunkShared {
  uint64_t scale_full[kScaleStages], scale_clean[kScaleStages], scale_empty[kScaleStages], k_full[4], k_empty[4], v_full[2], v_empty[2], half_full[2], half_empty[2];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2], o_empty[2], idle;
  uint32_t tmem;
  int there[kScaleStages];             // bit p: page p of the tile is there
  volatile int redo[kFlagRing];        // of the segment: f16 did not hold a value
  volatile int abort_code;
  int finished;                        // segments of this CTA whose results are written
  int asked_k, asked_v, asked_scales;  // loads that the producer has issued
};

// The row tile's positions, as every role sees them.
struct Seen {
  int any_low, any_high, all_low, all_high;
};
__device__ __forceinline__ Seen seen_by(const Cursor<kTile, kChunkRows>& at, int group, int window) {
  const int rows = at.rows(group), base = at.s.length - at.s.count, r0 = at.rt * kChunkRows;
  const int first = base + r0 / group, last = base + (r0 + rows - 1) / group;
  return {window > 0 ? max(first - window + 1, 0) : 0, last, window > 0 ? max(last - window + 1, 0) : 0, first};
}

// The unit's reference after a tile: 2^e above every finite scale of a position that is there and seen by any row; whole warp.
// Roles that need it follow it by themselves.
__device__ __forceinline__ int tile_exponent(const float* v_scale, int there, int position0, const Seen& seen, int lane) {
  const float4 v = reinterpret_cast<const float4*>(v_scale)[lane];
  const float x[4] = {v.x, v.y, v.z, v.w};
  unsigned top = 0u;
  const bool here = (there >> (lane / 16)) & 1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned bits = __float_as_uint(x[i]) & 0x7fffffffu;
    const int position = position0 + 4 * lane + i;
    if (here && position >= seen.any_low && position <= seen.any_high && bits < 0x7f800000u) top = max(top, bits);
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
__device__ __noinline__ void exact_row(const AttentionArgs& a, const KvSequence& s, int b, int head, int r, float* s_q, float* s_p) {
  const int lane = threadIdx.x % 32, t = r / a.group;
  const int position = s.length - s.count + t, low = a.window > 0 ? max(position - a.window + 1, 0) : 0;
  const long long column = static_cast<long long>(head * a.group + r % a.group) * D;
  const __nv_bfloat16* q = a.q + (s.first + t) * a.q_stride + column;
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
    *reinterpret_cast<__nv_bfloat162*>(a.out + (s.first + t) * a.out_stride + column + i * 64 + lane * 2) =
        __floats2bfloat162_rn(acc[2 * i] * inv, acc[2 * i + 1] * inv);
}

template <int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
attention_chunk_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ AttentionArgs a, int* __restrict__ status,
                       long long wait_limit) {
  using Shape = ChunkShape<D>;
  using Place = Cursor<kTile, kChunkRows>;
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
    for (int i = 0; i < kFlagRing; ++i) sh.redo[i] = 0;
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
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_bounded(bar, parity, &sh.abort_code, kStatusChunkTimeout, wait_limit); };

  // 512 threads at 128 registers are all there are: 256 of them at 64 leave 192 for each softmax thread, until the roles are done.
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    // ------------------------------------------------------------------------------------------ softmax, a thread per row
    const int slot = warp / 4, in_slot = tid % 128;
    const uint32_t lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t t_s = tmem + lanes + slot * 128, t_o = tmem + lanes + 256 + slot * 128;
    Place at;
    at.start(plan, s_plan);
    bool ok = true;
    int i = 0, tile_no = 0, segment_no = 0;     // of this slot
    for (int segment = 0; i < count; ++segment) {
      const int n = min(at.span.tiles - at.tile, count - i), rows = at.rows(a.group);
      const bool active = slot * 128 < rows, whole = n == at.span.tiles;
      const Seen seen = seen_by(at, a.group, a.window);
      const int row = slot * 128 + in_slot, r = at.rt * kChunkRows + row;
      const bool real = row < rows;
      const int token = real ? r / a.group : (at.rt * kChunkRows + rows - 1) / a.group;     // (rows beyond the last copy its bounds)
      const int high = at.s.length - at.s.count + token, low = a.window > 0 ? max(high - a.window + 1, 0) : 0;
      const __nv_bfloat16* const q = a.q + (at.s.first + token) * a.q_stride + (at.head * a.group + (real ? r % a.group : 0)) * D;
      float unit = 0.0f;
      if (active) {
        // ---- q as two e4m3 terms of q * 2^k, the row's largest at 2^7 .. 2^8
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
        const float up = copysignf(__int_as_float((k + 127) << 23), a.scale_log2);
        // (a scale of zero keeps a factor, so that -infinity stays what it is)
        unit = top >= 0x7f80u ? __int_as_float(0x7fffffff) : fmaxf(fabsf(a.scale_log2) * __int_as_float((127 - k) << 23), 1e-30f);
        uint8_t* const hi_tile = smem + Shape::kQ + 2 * slot * Shape::kTileBytes;
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
          const int to = swizzled<D>(in_slot, c);
          *reinterpret_cast<uint4*>(hi_tile + to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(hi_tile + Shape::kTileBytes + to) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_full[slot]);
      }
      const int warp_low = __reduce_max_sync(0xffffffffu, low), warp_high = __reduce_min_sync(0xffffffffu, high);   // seen by every row of the warp
      float m = -INFINITY;
      uint64_t l2 = 0ull;                       // two halves of the sum
      int exponent = -100;
      for (int j = 0; j < n; ++j, ++i) {
        const int ss = i % kScaleStages, position0 = (at.span.first + at.tile + j) * kTile;
        mbar_wait_or_clear(ok, &sh.scale_full[ss], i / kScaleStages & 1, &sh.abort_code, kStatusChunkTimeout, wait_limit);
        mbar_wait_or_clear(ok, &sh.scale_clean[ss], i / kScaleStages & 1, &sh.abort_code, kStatusChunkTimeout, wait_limit);
        if (active) {
          const float* const k_scale = reinterpret_cast<const float*>(smem + Shape::kScales) + ss * 2 * kTile;
          const int there = sh.there[ss];
          const int e = tile_exponent(k_scale + kTile, there, position0, seen, lane);
          float fade = 1.0f;
          if (j == 0) {
            exponent = e;
          } else if (e > exponent + kUnitGrowth) {
            fade = ex2(static_cast<float>(exponent - e));
            exponent = e;
          }
          mbar_wait_or_clear(ok, &sh.s_full[slot], tile_no & 1, &sh.abort_code, kStatusChunkTimeout, wait_limit);
          __syncwarp();
          tc_fence_after();
          uint32_t s[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(t_s + 32 * c, s[c]);
          tmem_ld_wait_for(s[0]);
#pragma unroll
          for (int c = 1; c < 4; ++c) tmem_landed(s[c]);
          // scores in units of the row's: times the key's scale
#pragma unroll
          for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int e4 = 0; e4 < 8; ++e4) {
              const float4 ks = *reinterpret_cast<const float4*>(k_scale + 32 * c + 4 * e4);
              float x0, x1, x2, x3;
              f32x2_unpack(f32x2_mul(f32x2_pack_bits(s[c][4 * e4], s[c][4 * e4 + 1]), f32x2_pack(ks.x, ks.y)), x0, x1);
              f32x2_unpack(f32x2_mul(f32x2_pack_bits(s[c][4 * e4 + 2], s[c][4 * e4 + 3]), f32x2_pack(ks.z, ks.w)), x2, x3);
              s[c][4 * e4] = __float_as_uint(x0);
              s[c][4 * e4 + 1] = __float_as_uint(x1);
              s[c][4 * e4 + 2] = __float_as_uint(x2);
              s[c][4 * e4 + 3] = __float_as_uint(x3);
            }
          }
          if (position0 < warp_low || position0 + kTile - 1 > warp_high || there != 3) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              // bit b: position position0 + 32 c + b is there and seen
              const int first = low - position0 - 32 * c, last = high - position0 - 32 * c;
              uint32_t bits = last < 0 || first > 31 || !(there >> (c / 2) & 1) ? 0u : 0xffffffffu;
              if (last >= 0 && last < 31) bits &= (2u << last) - 1u;
              if (first > 0 && first <= 31) bits &= 0xffffffffu << first;
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
            float l0, l1;
            f32x2_unpack(l2, l0, l1);
            l2 = f32x2_pack(l0 * f, l1 * f);
            m = top;
          }
          if (j > 0 && __any_sync(0xffffffffu, fade != 1.0f)) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(t_o + 32 * c, o);
              tmem_ld_wait_for(o);
#pragma unroll
              for (int b = 0; b < 32; ++b) o[b] = __float_as_uint(__uint_as_float(o[b]) * fade);
              tmem_st32(t_o + 32 * c, o);
            }
          }
          const float shift = kHeadroom - finite_or_zero(m);
          const uint64_t unit2 = f32x2_pack(unit, unit), shift2 = f32x2_pack(shift, shift);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t p[32];
#pragma unroll
            for (int b = 0; b < 32; ++b) {
              const int c = 2 * h + b / 16, at2 = b % 16 * 2;
              float x0, x1;
              f32x2_unpack(f32x2_fma(f32x2_pack_bits(s[c][at2], s[c][at2 + 1]), unit2, shift2), x0, x1);
              x0 = ex2(x0);
              x1 = ex2(x1);
              l2 = f32x2_add(l2, f32x2_pack(x0, x1));
              p[b] = pack_half2(x0, x1);
            }
            tmem_st32(t_s + 32 * h, p);
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_full[slot]);
          ++tile_no;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.scale_empty[ss]);
        if (!__all_sync(0xffffffffu, ok)) break;
      }
      // ---- the segment's end
      if (active) {
        mbar_wait_or_clear(ok, &sh.o_full[slot], segment_no & 1, &sh.abort_code, kStatusChunkTimeout, wait_limit);
        __syncwarp();
        tc_fence_after();
        ++segment_no;
      }
      if (softmax_bar_any(!ok)) break;          // all eight warps meet here whatever failed, and leave together
      const bool redo = sh.redo[segment % kFlagRing] != 0;
      if (tid == 0) sh.redo[(segment + kFlagRing - 1) % kFlagRing] = 0;     // the segment before: everybody has read it
      const long long unit_start = w0 + (i - n) - at.tile;
      const int slot_no = 2 * static_cast<int>(blockIdx.x) + (w0 >= unit_start ? 0 : 1);
      const long long part = static_cast<long long>(slot_no) * kChunkRows + row;
      if (active) {
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
            uint4* to = reinterpret_cast<uint4*>(a.out + (at.s.first + token) * a.out_stride + (at.head * a.group + r % a.group) * D + 32 * c);
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
            float4* to = reinterpret_cast<float4*>(a.partial + part * D + 32 * c);
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
      float* const s_q = reinterpret_cast<float*>(smem + Shape::kRedo) + warp * (D + kKvPage);
      if (whole) {
        if (redo)
          for (int x = warp; x < rows; x += 8) exact_row<D>(a, at.s, at.b, at.head, at.rt * kChunkRows + x, s_q, s_q + D);
      } else {
        const int first = piece_of(total, ctas, unit_start), last = piece_of(total, ctas, unit_start + at.span.tiles - 1);
        __threadfence();
        named_bar_sync(1, 256);
        if (tid == 0) {
          const bool is_last = atomicAdd(a.tickets + first, 1) == last - first;
          if (is_last) a.tickets[first] = 0;
          s_plan.last = is_last;
        }
        named_bar_sync(1, 256);
        if (s_plan.last) {
          __threadfence();
          const float4* stats = reinterpret_cast<const float4*>(a.partial + 2ll * ctas * kChunkRows * D);
          bool any_redo = false;
          for (int c = first; c <= last; ++c)
            any_redo |= __ldcg(stats + static_cast<long long>(2 * c + (piece_start(total, ctas, c) >= unit_start ? 0 : 1)) * kChunkRows).w != 0.0f;
          if (any_redo) {
            for (int x = warp; x < rows; x += 8) exact_row<D>(a, at.s, at.b, at.head, at.rt * kChunkRows + x, s_q, s_q + D);
          } else {
            join_parts<D, kChunkRows>(a, at.s, at.rt, at.head, rows, total, ctas, first, last, unit_start, tid, 256);
          }
        }
      }
      if (tid == 0) sh.finished = segment + 1;
      if (i < count) at.next_unit(plan);
    }
    asm volatile("setmaxnreg.dec.sync.aligned.u32 128;");
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (warp == 13) {
    // ------------------------------------------------------------------------------------------ loads
    if (lane == 0) {
      const uint64_t keep = l2_policy_evict_normal();      // other row tiles of the sequence read the same pages
      Place at;
      at.start(plan, s_plan);
      int entry[2];
      Seen seen = seen_by(at, a.group, a.window);
      auto entries = [&]() {                               // of the tile to ask for next: read one tile ahead
        const int32_t* table = a.batch.block_table + static_cast<long long>(at.b) * a.batch.max_pages;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int page = 2 * (at.span.first + at.tile) + p;
          entry[p] = page < a.batch.max_pages && page * kKvPage <= seen.any_high && (page + 1) * kKvPage > seen.any_low ? __ldg(table + page) : -1;
        }
      };
      entries();
      for (int i = 0; i < count; ++i) {
        const int ss = i % kScaleStages, ks = i % Shape::kKStages, vs = i % Shape::kVStages;
        int there = 0;
#pragma unroll
        for (int p = 0; p < 2; ++p) there |= (entry[p] >= 0 && entry[p] < a.cache.num_pages) << p;
        const int pages = (there & 1) + (there >> 1);
        if (!wait(&sh.scale_empty[ss], (i / kScaleStages & 1) ^ 1)) break;
        sh.there[ss] = there;
        mbar_arrive_expect_tx(&sh.scale_full[ss], pages * 2 * kKvPage * 4);
        float* const scales = reinterpret_cast<float*>(smem + Shape::kScales) + ss * 2 * kTile;
        const int head = at.head;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          if (!(there >> p & 1)) continue;
          bulk_load(scales + p * kKvPage, kv_block<D>(a.cache, entry[p], 0, head) + kKvPage * D, kKvPage * 4, &sh.scale_full[ss], keep);
          bulk_load(scales + kTile + p * kKvPage, kv_block<D>(a.cache, entry[p], 1, head) + kKvPage * D, kKvPage * 4, &sh.scale_full[ss], keep);
        }
        sh.asked_scales = i + 1;
        if (!wait(&sh.k_empty[ks], (i / Shape::kKStages & 1) ^ 1)) break;
        mbar_arrive_expect_tx(&sh.k_full[ks], pages * kKvPage * D);
#pragma unroll
        for (int p = 0; p < 2; ++p)
          if (there >> p & 1) tma_load_4d(smem + Shape::kK + ks * Shape::kTileBytes + p * kKvPage * D, &map, &sh.k_full[ks], 0, 0, head, entry[p], keep);
        sh.asked_k = i + 1;
        if (!wait(&sh.v_empty[vs], (i / Shape::kVStages & 1) ^ 1)) break;
        mbar_arrive_expect_tx(&sh.v_full[vs], pages * kKvPage * D);
#pragma unroll
        for (int p = 0; p < 2; ++p)
          if (there >> p & 1) tma_load_4d(smem + Shape::kV + vs * Shape::kTileBytes + p * kKvPage * D, &map, &sh.v_full[vs], 0, 0, a.cache.heads + head, entry[p], keep);
        sh.asked_v = i + 1;
        if (i + 1 < count) {
          if (++at.tile == at.span.tiles) {
            at.next_unit(plan);
            seen = seen_by(at, a.group, a.window);
          }
          entries();
        }
      }
    }
    __syncwarp();
  } else if (warp == 12) {
    // ------------------------------------------------------------------------------------------ MMAs
    if (lane == 0) {
      Place at;
      at.start(plan, s_plan);
      const uint32_t qk_desc = umma_idesc_e4m3_m128(kTile), pv_desc = umma_idesc_f16_m128_n_major(D);
      auto operand = [&](int offset) {
        return D == 128 ? umma_smem_desc_sw128(smem_u32(smem + offset)) : umma_smem_desc_sw64(smem_u32(smem + offset));
      };
      auto scores = [&](int slot, int ks) {
        const uint64_t k = operand(Shape::kK + ks * Shape::kTileBytes);
#pragma unroll
        for (int term = 0; term < 2; ++term) {
          const uint64_t q = operand(Shape::kQ + (2 * slot + term) * Shape::kTileBytes);
#pragma unroll
          for (int step = 0; step < D / 32; ++step) umma_f8(tmem + slot * 128, q + 2 * step, k + 2 * step, qk_desc, term + step > 0 ? 1u : 0u);
        }
        umma_commit(&sh.s_full[slot]);
      };
      auto values = [&](int slot, int hs, bool first) {
        const uint64_t v = umma_smem_desc_n_major_sw128(smem_u32(smem + Shape::kHalf + hs * Shape::kHalfBytes), kTile * 128);
#pragma unroll
        for (int step = 0; step < kTile / 16; ++step)
          umma_f16_ts(tmem + 256 + slot * 128, tmem + slot * 128 + 8 * step, v + 128 * step, pv_desc, first && step == 0 ? 0u : 1u);
      };
      int i = 0, tiles[2] = {0, 0}, segments[2] = {0, 0};  // tiles and segments of each slot so far
      bool alive = true;
      while (i < count && alive) {
        const int n = min(at.span.tiles - at.tile, count - i);
        const int slots = at.rows(a.group) > 128 ? 2 : 1;
        for (int s = 0; s < slots && alive; ++s) alive = wait(&sh.q_full[s], segments[s] & 1);
        alive = alive && wait(&sh.k_full[i % Shape::kKStages], i / Shape::kKStages & 1);
        if (!alive) break;
        tc_fence_after();
        for (int s = 0; s < slots; ++s) scores(s, i % Shape::kKStages);
        umma_commit(&sh.k_empty[i % Shape::kKStages]);
        for (int j = 0; j < n && alive; ++j) {
          const int now = i + j, next = now + 1;
          const bool more = j + 1 < n;
          if (more) alive = wait(&sh.k_full[next % Shape::kKStages], next / Shape::kKStages & 1);
          alive = alive && wait(&sh.half_full[now % 2], now / 2 & 1);
          for (int s = 0; s < slots && alive; ++s) {
            if (j == 0) alive = wait(&sh.o_empty[s], (segments[s] & 1) ^ 1);
            alive = alive && wait(&sh.p_full[s], tiles[s] & 1);
            if (!alive) break;
            tc_fence_after();
            values(s, now % 2, j == 0);
            ++tiles[s];
            if (s + 1 == slots) umma_commit(&sh.half_empty[now % 2]);
            if (more) scores(s, next % Shape::kKStages);
            else umma_commit(&sh.o_full[s]);
          }
          if (alive && more) umma_commit(&sh.k_empty[next % Shape::kKStages]);
        }
        for (int s = 0; s < slots; ++s) ++segments[s];
        i += n;
        if (i < count) at.next_unit(plan);
      }
    }
    __syncwarp();
  } else if (warp >= 8 && warp < 12) {
    // ------------------------------------------------------------------------------------------ values to f16, a thread per position
    const int t = tid - 8 * 32;
    Place at;
    at.start(plan, s_plan);
    bool ok = true;
    int segment = 0, unit = -100;
    bool fresh = true;
    Seen seen = seen_by(at, a.group, a.window);
    for (int i = 0; i < count; ++i) {
      const int ss = i % kScaleStages, vs = i % Shape::kVStages, hs = i % 2;
      mbar_wait_or_clear(ok, &sh.scale_full[ss], i / kScaleStages & 1, &sh.abort_code, kStatusChunkTimeout, wait_limit);
      float* const k_scale = reinterpret_cast<float*>(smem + Shape::kScales) + ss * 2 * kTile;
      const float* const v_scale = k_scale + kTile;
      const int there = sh.there[ss], position0 = (at.span.first + at.tile) * kTile;
      const int e = tile_exponent(v_scale, there, position0, seen, lane);
      if (fresh || e > unit + kUnitGrowth) unit = e;
      fresh = false;
      const float scale = v_scale[t];
      const bool valid = (there >> (t / kKvPage) & 1) && position0 + t >= seen.any_low && position0 + t <= seen.any_high;
      const bool mixed = position0 < seen.all_low || position0 + kTile - 1 > seen.all_high;     // some rows may see what others do not
      const float r = scale * __int_as_float((kUnitShift - unit + 127) << 23);
      // r as two f16 terms, so that the product with a byte's value is rounded once
      const __half hi = __float2half_rn(r);
      const __half2 r_hi = __half2half2(hi), r_lo = __half2half2(__float2half_rn(r - __half2float(hi)));
      mbar_wait_or_clear(ok, &sh.v_full[vs], i / Shape::kVStages & 1, &sh.abort_code, kStatusChunkTimeout, wait_limit);
      const uint8_t* const from = smem + Shape::kV + vs * Shape::kTileBytes;
      // Zero times NaN is NaN: where some rows see a value that is not finite and others do not, its bytes become zeros and the NaN
      // goes by way of its score to the rows that see it.
      bool bad = false;
      if (mixed && valid) {
        uint32_t over = 0u;
#pragma unroll 4
        for (int chunk = 0; chunk < D / 16; ++chunk) {
          const uint4 p = *reinterpret_cast<const uint4*>(from + swizzled<D>(t, chunk));
          over |= ((p.x & 0x7f7f7f7fu) + 0x01010101u) | ((p.y & 0x7f7f7f7fu) + 0x01010101u) | ((p.z & 0x7f7f7f7fu) + 0x01010101u) | ((p.w & 0x7f7f7f7fu) + 0x01010101u);
        }
        bad = (over & 0x80808080u) != 0u || !(fabsf(scale) <= 3.402823466e38f);
        if (bad) k_scale[t] = __int_as_float(0x7fffffff);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.scale_clean[ss]);
      mbar_wait_or_clear(ok, &sh.half_empty[hs], (i / 2 & 1) ^ 1, &sh.abort_code, kStatusChunkTimeout, wait_limit);
      uint8_t* const to = smem + Shape::kHalf + hs * Shape::kHalfBytes + t * 128;
      if (valid && !bad) {
        uint32_t any = 0u;
#pragma unroll 4
        for (int chunk = 0; chunk < D / 16; ++chunk) {
          const uint4 p = *reinterpret_cast<const uint4*>(from + swizzled<D>(t, chunk));
          const uint32_t w[4] = {p.x, p.y, p.z, p.w};
          uint32_t h[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t bits = e4m3x2_to_half2(w[j / 2] >> (16 * (j % 2)));
            const __half2 v = *reinterpret_cast<const __half2*>(&bits);
            const __half2 y = __hfma2(v, r_hi, __hmul2(v, r_lo));
            h[j] = *reinterpret_cast<const uint32_t*>(&y);
          }
          any |= (p.x | p.y | p.z | p.w) & 0x7f7f7f7fu;
          uint8_t* const row = to + chunk / 4 * (kTile * 128);
          *reinterpret_cast<uint4*>(row + (((2 * chunk) % 8 ^ (t & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint4*>(row + (((2 * chunk + 1) % 8 ^ (t & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
        }
        if (any != 0u && fabsf(r) < kSmallestUnit) sh.redo[segment % kFlagRing] = 1;
      } else {
#pragma unroll 4
        for (int chunk = 0; chunk < D / 8; ++chunk) *reinterpret_cast<uint4*>(to + chunk / 8 * (kTile * 128) + chunk % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sh.half_full[hs]);
        mbar_arrive(&sh.v_empty[vs]);
        mbar_arrive(&sh.scale_empty[ss]);
      }
      if (!__all_sync(0xffffffffu, ok)) break;
      if (i + 1 < count && ++at.tile == at.span.tiles) {
        at.next_unit(plan);
        seen = seen_by(at, a.group, a.window);
        ++segment;
        fresh = true;
      }
    }
    }
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
    Place at;
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
          const int first = piece_of(total, ctas, unit_start), last = piece_of(total, ctas, unit_start + at.span.tiles - 1);
          __threadfence();
          __syncthreads();
          if (tid == 0) {
            const bool is_last = atomicAdd(a.tickets + first, 1) == last - first;
            if (is_last) a.tickets[first] = 0;
            s_plan.last = is_last;
          }
          __syncthreads();
          if (s_plan.last) {
            __threadfence();
            join_parts<D, kChunkRows>(a, at.s, at.rt, at.head, rows, total, ctas, first, last, unit_start, tid, kChunkThreads);
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
