// Attention of new tokens over the paged KV cache in 4 bits (include/syfi_kv4.h).
//
//   x_j = scale * kscale_j * sum_d q_d k_jd,   out_d = sum_j exp(x_j) vscale_j v_jd / sum_j exp(x_j)   over the visible positions j
// in one pass over the cache, k and v being code * group scale, which f16 holds exactly (at most 6 * 448, two bits times four).  With x in
// units of log2 and references m (of the sum l) and n (of the sum o) that follow the largest terms,
//   l = sum 2^(x_j - m),   o_d = sum 2^(x_j + log2 vscale_j - n) v_jd,   out_d = o_d 2^(n - m) / l.
#include <cstdio>
#include <mutex>

#include "kv4_chunk.cuh"
#include "stream_scratch.h"

namespace syfi {

namespace {

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The transpose of an 8 x 8 matrix of f16: lane 4 i + j has elements (i, 2 j) and (i, 2 j + 1) before, (2 j, i) and (2 j + 1, i) after.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t lo, uint32_t hi) { return e4m3x2_to_half2(lo | hi << 8); }
// Each half twice.  (Moves of halves: a multiplication can take either half of a register for both, where a byte permutation costs an
// instruction; 32 sequences of 65536 positions 284 us instead of 290.)
__device__ __forceinline__ void both_halves(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tmov.b32 %0, {a, a};\n\tmov.b32 %1, {b, b};\n\t}" : "=r"(lo), "=r"(hi) : "r"(v));
}

// ---------------------------------------------------------------- few rows per sequence and key head: decoding
// A CTA walks its piece of the pages.  A warp has every fourth page to itself, so that no warp waits for another before the end of a unit, for
// 8 NT rows.  A page's two blocks come by two bulk copies into a ring of stages: the warp that has used up a stage asks for the page that
// goes there next, whichever warp's that is.  mma.sync m16n8k16 in f16, whose big operand the lanes make from the codes in registers,
// so that a row tile is as narrow as an MMA allows:
//   scores:  positions (M) x rows (N) = K Q^T.  A lane has one group of 16 dimensions of two positions in each plane, whose scale it
//            multiplies in; the MMAs' k index permutes the dimensions, alike in q.
//   values:  dimensions (M) x rows (N) = V^T P^T.  A lane pairs the codes of two positions, a byte for each dimension; its D / 8 dimensions
//            have one group scale.  The weights come from the scores' layout by an 8 x 8 transpose (movmatrix).
// Which position an index of the scores stands for is chosen so that both reads of the rows of 32 bytes are free of bank conflicts: index i
// of eight is position i ^ (i >> 2 & 1).
//
// What bounds it is the latency of a page's steps with three warps to a scheduler: 1221 instructions of a warp for 64 positions of 128
// dimensions, a third of them conversions, which issue at half a clock's rate, take 60 % of the issue slots, and the warps' conversions, MMAs and
// exponentials overlap one another's no further.  32 sequences of 65536 positions, 4 key heads: 252 to 264 us, where the loads alone take
// 210 and the bytes 195 at the rate of a copy; with heads of 64 170.  Three blocks of 168 registers to an SM; four of 128: 264.  With 16 rows
// (two blocks of 255 registers, two of them in local memory for a while: 16 bytes) a page's conversions serve twice the rows.
//
// kDecodeExtra is what a unit costs besides its pages, in pages: the prologue, its end, the join.  With 3, 6 and 9: 24 sequences of 300 to 30000
// positions with 8 key heads 64, 58 and 58 us (8 rows), 98, 83 and 80 (16 rows), with heads of 64 47, 42 and 41 (4 rows), 74, 62 and 58
// (16 rows); 200 sequences of 100 to 3000 positions, heads of 64, 64, 55 and 56.
constexpr int kDecodeExtra = 6;
constexpr float kFarBehind = 1.2676506e30f;   // 2^100 between the references of the two sums: the values' follows
constexpr int kWarps = 4;
constexpr int kStatusTimeout = 401;

template <int D, int NT>
struct Decode4Shape {
  static constexpr int kRows = 8 * NT;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kBlocks = NT == 1 ? 3 : 2;          // per SM
  static constexpr int kStageBytes = 2 * Kv4Block<D>::kBytes;
  static constexpr int kMerge = 2 * 8 * NT * D * 4;        // bytes
  static constexpr int kRoom = (NT == 1 ? 74 : 110) * 1024 - kMerge;
  static constexpr int kStages = kRoom / kStageBytes < 12 ? kRoom / kStageBytes : 12;
  static constexpr int kSmem = kStages * kStageBytes + kMerge;
};

// How far the loads of a warp have come: pages `tile`, `tile` + 4, ... below `end` of a segment.
struct LoadWalk {
  const int32_t* table;                // of the segment's sequence, from the unit's first page on
  int tile, end, head;
};

template <int D, int NT>
struct DecodeShared {
  using Walk = Cursor<kKvPage, 8 * NT, kDecodeExtra>;
  PlanShared plan;
  uint64_t full[Decode4Shape<D, NT>::kStages];
  int there[Decode4Shape<D, NT>::kStages];
  volatile int holds[Decode4Shape<D, NT>::kStages];   // number of the page that a stage was last asked for
  Walk load[kWarps];                   // the segment that a warp's loads are in
  int skip[kWarps];                    // pages from its beginning to the warp's first there
  float4 stat[kWarps][8 * NT];
  volatile int failed;                 // a copy did not arrive in time
};

// Waits for a page's copies, at most `limit` SM clocks, and not once another warp has waited in vain.  Warps drift apart, and a phase's parity
// says only which of two it is: so first the stage must have been asked for this very page (`holds`), which it is when the page in front of it
// has been used up.  With a limit of one clock nothing counts as there in time: pages are nearly always there before they are asked about, and
// a test of what follows must not depend on it.
__device__ __forceinline__ bool landed(uint64_t* bar, uint32_t parity, const volatile int* holds, int page, volatile int* failed, long long limit) {
  if (*holds == page && limit > 1 && mbar_try_wait(bar, parity)) return true;
  const long long begun = clock64();
  do {
    if (*failed != 0) return false;
    if (clock64() - begun > limit) {
      *failed = 1;
      return false;
    }
  } while (*holds != page || !mbar_try_wait(bar, parity));
  return true;
}

template <int D, int NT>
__global__ void __launch_bounds__(Decode4Shape<D, NT>::kThreads, Decode4Shape<D, NT>::kBlocks)
kv4_decode_kernel(const __grid_constant__ AttentionArgs a, int* __restrict__ status, long long wait_limit) {
  using Shape = Decode4Shape<D, NT>;
  using Walk = Cursor<kKvPage, Shape::kRows, kDecodeExtra>;
  using Block = Kv4Block<D>;
  constexpr int kRows = Shape::kRows, kStages = Shape::kStages, kPlanes = D / 64, kSteps = D / 16, kMmas = D / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ DecodeShared<D, NT> sh;
  float* const s_merge = reinterpret_cast<float*>(smem + kStages * Shape::kStageBytes);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, c = lane % 4;

  pdl_wait();
  pdl_trigger();
  const Plan<kKvPage, kRows, kDecodeExtra> plan = {a.batch, a.cache.heads, a.group, a.window};
  const long long total = plan.total(sh.plan);
  const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
  if (static_cast<int>(blockIdx.x) >= ctas) return;
  const long long w0 = piece_start(total, ctas, blockIdx.x), w1 = piece_start(total, ctas, blockIdx.x + 1);
  if (tid < kStages) {
    mbar_init(&sh.full[tid], 1);
    sh.holds[tid] = -1;
    fence_barrier_init();
  }
  if (tid == 0) sh.failed = 0;
  plan.locate(sh.plan, w0);                  // (ends with a barrier)

  Walk use;
  use.start(plan, sh.plan, static_cast<int>(w1 - w0));
  if (use.left <= 0) return;
  // Pages of the piece are numbered: page p is warp p % 4's, in stage p % kStages.
  if (lane == 0) {
    sh.load[warp] = use;
    sh.skip[warp] = warp;
  }
  __syncwarp();
  LoadWalk walk = {nullptr, 0, 0, 0};
  int entry = -1;                            // of the page to ask for next: read one page ahead
  bool more = true;
  // On to the walk's page, of the next segment that has any of this warp's.
  auto settle = [&]() {
    if (walk.tile >= walk.end) {
      if (lane == 0) {
        Walk& at = sh.load[warp];
        int skip = sh.skip[warp];
        while (at.left > 0 && skip >= at.tiles_here()) {
          const int n = at.tiles_here();
          skip -= n;
          at.advance(plan, n);
        }
        // (this lane's walk goes on behind the segment: skip counts from its end)
        if (at.left > 0) {
          const int n = at.tiles_here();
          sh.skip[warp] = skip + (n - skip + kWarps - 1) / kWarps * kWarps - n;
          walk = {a.batch.block_table + static_cast<long long>(at.b) * a.batch.max_pages + at.span.first, at.tile + skip, at.tile + n, at.head};
          at.advance(plan, n);
        } else {
          walk.head = -1;
        }
      }
      walk.table = reinterpret_cast<const int32_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(walk.table), 0));
      walk.tile = __shfl_sync(0xffffffffu, walk.tile, 0);
      walk.end = __shfl_sync(0xffffffffu, walk.end, 0);
      walk.head = __shfl_sync(0xffffffffu, walk.head, 0);
      more = walk.head >= 0;
    }
    if (more) entry = __ldg(walk.table + walk.tile);
  };
  auto ask = [&](int stage, int page) {
    if (!more) return;
    if (lane == 0) {
      const bool there = entry >= 0 && entry < a.cache.num_pages;
      sh.there[stage] = there;
      sh.holds[stage] = page;
      if (there) {
        mbar_arrive_expect_tx(&sh.full[stage], Shape::kStageBytes);
        uint8_t* const to = smem + stage * Shape::kStageBytes;
        const uint64_t once = l2_policy_evict_first();       // (32 sequences of 65536 positions 256 us instead of 262)
        bulk_load(to, kv4_block<D>(a.cache, entry, 0, walk.head), Block::kBytes, &sh.full[stage], once);
        bulk_load(to + Block::kBytes, kv4_block<D>(a.cache, entry, 1, walk.head), Block::kBytes, &sh.full[stage], once);
      } else {
        mbar_arrive(&sh.full[stage]);
      }
    }
    walk.tile += kWarps;
    settle();
  };
  settle();
  // A warp asks for the pages that follow its own by a round of stages, so at first for its own among the first kStages, then for those.
  constexpr int kFirst = kStages / kWarps;   // whole rounds of warps among the first stages
#pragma unroll
  for (int i = 0; i < kFirst; ++i) ask(i * kWarps + warp, i * kWarps + warp);
  if constexpr (kStages % kWarps != 0) {
    if (warp < kStages % kWarps) ask(kFirst * kWarps + warp, kFirst * kWarps + warp);
    // Page p + kStages is warp (p + kStages) % 4's: from here on this warp's walk is that of another, which has just asked for its first ones.
    __syncthreads();
    const int other = (warp + kStages) % kWarps;
    const Walk its_load = sh.load[other];
    const int its_skip = sh.skip[other];
    LoadWalk* const hand = reinterpret_cast<LoadWalk*>(s_merge);
    int* const hand_entry = reinterpret_cast<int*>(hand + kWarps);
    if (lane == 0) {
      hand[warp] = walk;
      hand_entry[2 * warp] = entry;
      hand_entry[2 * warp + 1] = more;
    }
    __syncthreads();
    walk = hand[other];
    entry = hand_entry[2 * other];
    more = hand_entry[2 * other + 1] != 0;
    if (lane == 0) {
      sh.load[warp] = its_load;
      sh.skip[warp] = its_skip;
    }
    __syncthreads();
  }
  int page0 = 0;                             // number of the segment's first page
  int stage = warp % kStages;                // of this warp's next page, and the parity of its use
  uint32_t parity = 0;
  bool lost = false;                         // a page of this warp did not come in time
  static_assert(kStages >= kWarps, "a stage for every warp's page");

  // This lane's positions of each 16: t0 and t0 + 8; its rows of the scores: 8 t + 2 c and 8 t + 2 c + 1.
  const int t0 = g ^ (g >> 2 & 1), v0 = (2 * c) ^ (c >> 1), v1 = (2 * c + 1) ^ (c >> 1);
  uint32_t qb[NT][kSteps][2];
  // Of each row: what a score is worth; the reference of this lane's sum, and the sum; the reference of the values' sum, and 2^(m - n + 7).
  float unit[NT][2], m[NT][2], l[NT][2], n[NT][2], up[NT][2], o[NT][kMmas][4];
  int low[NT][2], high[NT][2];               // positions that the rows see

  while (use.left > 0) {
    // ---- a segment: what this piece has of a unit
    const int tiles = use.tiles_here(), rows = use.rows(a.group), base = use.s.length - use.s.count, r0 = use.rt * kRows;
    const int first = base + r0 / a.group, last = base + (r0 + rows - 1) / a.group;
    const int all_low = a.window > 0 ? max(last - a.window + 1, 0) : 0, any_low = a.window > 0 ? max(first - a.window + 1, 0) : 0;
    const int all_high = first, any_high = last;         // positions that all / any of the unit's rows see
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      // 2^k that brings the row's largest magnitude to 2^14 .. 2^15: f16 then holds bf16 values exactly down to 2^-29 of it
      const int row = t * 8 + g, r = r0 + row;
      const bool real = row < rows;
      const __nv_bfloat16* from = a.q + (use.s.first + (real ? r / a.group : 0)) * a.q_stride + (use.head * a.group + (real ? r % a.group : 0)) * D;
      uint2 raw[kSteps];
      unsigned top = 0u;
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
        raw[step] = real ? __ldg(reinterpret_cast<const uint2*>(from + 64 * (step / 4) + 16 * c + 4 * (step % 4))) : make_uint2(0u, 0u);
        top = max(max(top, raw[step].x & 0x7fffu), (raw[step].x >> 16) & 0x7fffu);
        top = max(max(top, raw[step].y & 0x7fffu), (raw[step].y >> 16) & 0x7fffu);
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int k = top == 0u ? 0 : min(14 - (static_cast<int>(top >> 7) - 127), 120);
      const float factor = __int_as_float((k + 127) << 23);
      const float worth = top >= 0x7f80u ? __int_as_float(0x7fffffff) : a.scale_log2 * __int_as_float((127 - k) << 23);
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
        qb[t][step][0] = pack_half2(__uint_as_float(raw[step].x << 16) * factor, __uint_as_float(raw[step].x & 0xffff0000u) * factor);
        qb[t][step][1] = pack_half2(__uint_as_float(raw[step].y << 16) * factor, __uint_as_float(raw[step].y & 0xffff0000u) * factor);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        unit[t][i] = __shfl_sync(0xffffffffu, worth, 8 * c + 4 * i);
        const int mine = t * 8 + 2 * c + i;
        const int position = base + (mine < rows ? (r0 + mine) / a.group : 0);
        low[t][i] = a.window > 0 ? max(position - a.window + 1, 0) : 0;
        high[t][i] = mine < rows ? position : -1;
        m[t][i] = n[t][i] = -INFINITY;
        l[t][i] = up[t][i] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < kMmas; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][j][e] = 0.0f;
    }

    const int begin = (warp - page0) & (kWarps - 1);
    for (int tile = begin; tile < tiles; tile += kWarps) {
      if (lost || !__all_sync(0xffffffffu, landed(&sh.full[stage], parity, &sh.holds[stage], page0 + tile, &sh.failed, wait_limit))) {
        // Not in time, for this warp or another: the rows become NaN, and nothing more is asked for, since the stage may still be written.
        lost = true;
        more = false;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            l[t][i] = __int_as_float(0x7fffffff);
            n[t][i] = 0.0f;
          }
        break;
      }
      uint8_t* const keys = smem + stage * Shape::kStageBytes;
      uint8_t* const values = keys + Block::kBytes;
      float* const k_scale = reinterpret_cast<float*>(keys + Block::kScales);
      float* const v_scale = reinterpret_cast<float*>(values + Block::kScales);
      const int position0 = (use.span.first + use.tile + tile) * kKvPage;
      const bool plain = position0 >= all_low && position0 + kKvPage - 1 <= all_high;    // every row sees every position
      if (sh.there[stage]) {
        if (!plain) {
          // What a row does not see must not reach its sums, and zero times NaN is NaN: values of positions that no row sees become zeros,
          // and where some rows see a value that is not finite, the NaN goes by way of its score to those rows alone.  (Codes are always
          // finite.)
#pragma unroll
          for (int at = lane; at < kKvPage; at += 32) {
            uint32_t* const groups = reinterpret_cast<uint32_t*>(values + Block::kGroups) + at * (D / 64);
            uint32_t over = 0u;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) over |= (groups[i] & 0x7f7f7f7fu) + 0x01010101u;
            const bool bad = (over & 0x80808080u) != 0u || !(fabsf(v_scale[at]) <= 3.402823466e38f);
            if (bad || position0 + at < any_low || position0 + at > any_high) {
#pragma unroll
              for (int i = 0; i < D / 64; ++i) groups[i] = 0u;
              v_scale[at] = 1.0f;
              if (bad) k_scale[at] = __int_as_float(0x7fffffff);
            }
          }
          fence_proxy_async_smem();          // in front of the copy that comes here next
          __syncwarp();
        }
        float x[4][NT][4];                   // element e of block b: position 16 b + t0 + 8 (e / 2), row 2 c + e % 2
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          float part[kPlanes][NT][4];        // chains of MMAs
#pragma unroll
          for (int p = 0; p < kPlanes; ++p) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) part[p][t][e] = 0.0f;
            const uint2 w = *reinterpret_cast<const uint2*>(keys + p * kKv4Plane + (16 * b + t0) * 32 + c * 8);
            const uint2 v = *reinterpret_cast<const uint2*>(keys + p * kKv4Plane + (16 * b + t0 + 8) * 32 + c * 8);
            const uint8_t* const group = keys + Block::kGroups + (16 * b + t0) * kSteps + 4 * p + c;
            uint32_t sw, sv;
            both_halves(e4m3_pair(group[0], group[8 * kSteps]), sw, sv);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t wi = i < 2 ? w.x : w.y, vi = i < 2 ? v.x : v.y;
              const uint32_t ka[4] = {hmul2_bits(i % 2 ? e2m1x2_to_half2<2>(wi) : e2m1x2_to_half2<0>(wi), sw), hmul2_bits(i % 2 ? e2m1x2_to_half2<2>(vi) : e2m1x2_to_half2<0>(vi), sv),
                                      hmul2_bits(i % 2 ? e2m1x2_to_half2<3>(wi) : e2m1x2_to_half2<1>(wi), sw), hmul2_bits(i % 2 ? e2m1x2_to_half2<3>(vi) : e2m1x2_to_half2<1>(vi), sv)};
#pragma unroll
              for (int t = 0; t < NT; ++t) mma_f16(part[p][t], ka, qb[t][4 * p + i][0], qb[t][4 * p + i][1]);
            }
          }
          const float ks[2] = {k_scale[16 * b + t0], k_scale[16 * b + t0 + 8]};
          const float zero[2] = {ks[0] - ks[0], ks[1] - ks[1]};      // or NaN: a score that is minus infinity would count as not seen
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float sum = part[0][t][e];
              if constexpr (kPlanes == 2) sum += part[1][t][e];
              x[b][t][e] = fmaf(sum, ks[e / 2] * unit[t][e % 2], zero[e / 2]);
            }
        }
        if (!plain) {
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int position = position0 + 16 * b + t0 + 8 * (e / 2);
                if (position < low[t][e % 2] || position > high[t][e % 2]) x[b][t][e] = -INFINITY;
              }
        }
        bool grown = false, late = false;
        float top[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            top[t][i] = fmaxf(x[0][t][i], x[0][t][2 + i]);
#pragma unroll
            for (int b = 1; b < 4; ++b) top[t][i] = fmaxf(top[t][i], fmaxf(x[b][t][i], x[b][t][2 + i]));
            grown |= top[t][i] > m[t][i] + kSumGrowth;
          }
        if (__any_sync(0xffffffffu, grown)) {
          // a row's sum in this lane follows its scores once they are 2^16 above the reference; the lanes meet at the unit's end
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (top[t][i] > m[t][i] + kSumGrowth) {
                l[t][i] *= ex2(m[t][i] - top[t][i]);
                m[t][i] = top[t][i];
                up[t][i] = n[t][i] == -INFINITY ? 0.0f : ex2(top[t][i] - n[t][i] + kHeadroom);
                late |= up[t][i] > kFarBehind;
              }
            }
        }
        // weights, then those times the values' scales
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const float vs[2] = {v_scale[16 * b + t0], v_scale[16 * b + t0 + 8]};
#pragma unroll
          for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[b][t][e] = ex2(x[b][t][e] - finite_or_zero(m[t][e % 2]));
            l[t][0] += x[b][t][0] + x[b][t][2];
            l[t][1] += x[b][t][1] + x[b][t][3];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[b][t][e] *= vs[e / 2];
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            top[t][i] = fmaxf(x[0][t][i], x[0][t][2 + i]);
#pragma unroll
            for (int b = 1; b < 4; ++b) top[t][i] = fmaxf(top[t][i], fmaxf(x[b][t][i], x[b][t][2 + i]));
            late |= top[t][i] * up[t][i] > 32768.0f || (up[t][i] == 0.0f && top[t][i] > 0.0f);
          }
        if (__any_sync(0xffffffffu, late)) {
          // the reference of the values' sum follows, in all lanes of a row alike
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            float fade[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float most = m[t][i] + fmaxf(lg2(top[t][i]), -90.0f);      // (never further behind: a value may be zero)
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
              fade[i] = 1.0f;
              if (most > n[t][i] + kGrowth) {
                fade[i] = ex2(n[t][i] - most);
                n[t][i] = most;
              }
              up[t][i] = n[t][i] == -INFINITY || m[t][i] == -INFINITY ? 0.0f : ex2(m[t][i] - n[t][i] + kHeadroom);
            }
#pragma unroll
            for (int j = 0; j < kMmas; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[t][j][e] *= fade[e % 2];
          }
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          uint32_t pb[NT][2];
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) pb[t][u] = transposed(pack_half2(x[b][t][2 * u] * up[t][0], x[b][t][2 * u + 1] * up[t][1]));
          uint32_t even[2][D / 64], odd[2][D / 64], scale[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int at0 = 16 * b + 8 * u + v0, at1 = 16 * b + 8 * u + v1;
            const uint8_t* const groups = values + Block::kGroups + (D == 128 ? g : g / 2);
            scale[u] = e4m3_pair(groups[at0 * kSteps], groups[at1 * kSteps]);
            if constexpr (D == 128) {
              const uint8_t* const plane = values + g / 4 * kKv4Plane + g % 4 * 8;
              const uint2 w = *reinterpret_cast<const uint2*>(plane + at0 * 32), r = *reinterpret_cast<const uint2*>(plane + at1 * 32);
              even[u][0] = w.x; even[u][1] = w.y;
              odd[u][0] = r.x; odd[u][1] = r.y;
            } else {
              even[u][0] = *reinterpret_cast<const uint32_t*>(values + at0 * 32 + g * 4);
              odd[u][0] = *reinterpret_cast<const uint32_t*>(values + at1 * 32 + g * 4);
            }
          }
#pragma unroll
          for (int w = 0; w < D / 64; ++w) {
            // bytes that hold one dimension of both positions: dimensions 2 i, and 2 i + 1, of the word's eight
            uint32_t first_dims[2], second_dims[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              first_dims[u] = (even[u][w] & 0x0f0f0f0fu) | (odd[u][w] << 4 & 0xf0f0f0f0u);
              second_dims[u] = (even[u][w] >> 4 & 0x0f0f0f0fu) | (odd[u][w] & 0xf0f0f0f0u);
            }
            auto product = [&](auto byte) {
              constexpr int kByte = decltype(byte)::value;
              const uint32_t va[4] = {hmul2_bits(e2m1x2_to_half2<kByte>(first_dims[0]), scale[0]), hmul2_bits(e2m1x2_to_half2<kByte>(second_dims[0]), scale[0]),
                                      hmul2_bits(e2m1x2_to_half2<kByte>(first_dims[1]), scale[1]), hmul2_bits(e2m1x2_to_half2<kByte>(second_dims[1]), scale[1])};
#pragma unroll
              for (int t = 0; t < NT; ++t) mma_f16(o[t][4 * w + kByte], va, pb[t][0], pb[t][1]);
            };
            product(std::integral_constant<int, 0>{});
            product(std::integral_constant<int, 1>{});
            product(std::integral_constant<int, 2>{});
            product(std::integral_constant<int, 3>{});
          }
        }
      }
      __syncwarp();
      ask(stage, page0 + tile + kStages);
      stage += kWarps;
      if (stage >= kStages) {
        stage -= kStages;
        parity ^= 1u;
      }
    }
    page0 += tiles;

    // ---- the segment's end: lanes, then the four warps, then the unit's other pieces
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top = m[t][i];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        float sum = l[t][i] * ex2(m[t][i] - finite_or_zero(top));
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (g == 0) sh.stat[warp][8 * t + 2 * c + i] = make_float4(top, sum, n[t][i], 0.0f);
      }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float f[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float m_all = -INFINITY, n_all = -INFINITY, l_all = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          m_all = fmaxf(m_all, sh.stat[w][8 * t + 2 * c + i].x);
          n_all = fmaxf(n_all, sh.stat[w][8 * t + 2 * c + i].z);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 st = sh.stat[w][8 * t + 2 * c + i];
          l_all += st.y * ex2(st.x - finite_or_zero(m_all));
        }
        f[i] = ex2(n[t][i] - finite_or_zero(n_all));
        m[t][i] = m_all;
        n[t][i] = n_all;
        l[t][i] = l_all;
      }
#pragma unroll
      for (int j = 0; j < kMmas; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][j][e] *= f[e % 2];
    }
    float* const mine = s_merge + (warp & 1) * 8 * NT * D + lane;
    if (warp >= 2) {
#pragma unroll
      for (int k = 0; k < NT * kMmas * 4; ++k) mine[k * 32] = o[k / (kMmas * 4)][k / 4 % kMmas][k % 4];
    }
    __syncthreads();
    if (warp < 2) {
#pragma unroll
      for (int k = 0; k < NT * kMmas * 4; ++k) o[k / (kMmas * 4)][k / 4 % kMmas][k % 4] += mine[k * 32];
      if (warp == 1) {
#pragma unroll
        for (int k = 0; k < NT * kMmas * 4; ++k) mine[k * 32] = o[k / (kMmas * 4)][k / 4 % kMmas][k % 4];
      }
    }
    __syncthreads();
    const bool whole = tiles == use.span.tiles;
    const long long unit_start = w1 - use.left - use.tile;      // the place of its first page
    if (warp == 0) {
      const float* other = s_merge + 8 * NT * D + lane;
      const int slot = 2 * static_cast<int>(blockIdx.x) + (w0 >= unit_start ? 0 : 1);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = t * 8 + 2 * c + i, r = r0 + row;
          if (row >= rows) continue;
          float v[D / 8];                  // this lane's dimensions of the row, g * D / 8 and on
#pragma unroll
          for (int j = 0; j < kMmas; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) v[2 * j + e] = o[t][j][2 * e + i] + other[((t * kMmas + j) * 4 + 2 * e + i) * 32];
          if (whole) {
            const float f = l[t][i] == 0.0f || n[t][i] == -INFINITY ? 0.0f : ex2(n[t][i] - finite_or_zero(m[t][i]) - kHeadroom) / l[t][i];
            uint4* to = reinterpret_cast<uint4*>(a.out + (use.s.first + r / a.group) * a.out_stride + (use.head * a.group + r % a.group) * D + g * (D / 8));
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[8 * j + 2 * e] * f, v[8 * j + 2 * e + 1] * f);
                w[e] = *reinterpret_cast<const uint32_t*>(&h);
              }
              to[j] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
            const long long at = static_cast<long long>(slot) * kRows + row;
            float4* to = reinterpret_cast<float4*>(a.partial + at * D + g * (D / 8));
#pragma unroll
            for (int j = 0; j < D / 32; ++j) to[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            if (g == 0) reinterpret_cast<float4*>(a.partial + 2ll * ctas * kRows * D)[at] = make_float4(m[t][i], l[t][i], n[t][i], 0.0f);
          }
        }
    }
    if (!whole) {
      const Parts parts(total, ctas, unit_start, use.span.tiles);
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const bool is_last = atomicAdd(a.tickets + parts.first, 1) == parts.last - parts.first;
        if (is_last) a.tickets[parts.first] = 0;
        sh.plan.last = is_last;
      }
      __syncthreads();
      if (sh.plan.last) {
        __threadfence();
        join_parts<D, kRows>(a, use.s.first, r0, use.head, rows, ctas, parts, warp, 4);
      }
    }
    use.advance(plan, tiles);
  }
  if (sh.failed != 0) {
    // Copies may still be on their way: this CTA's memory must not be the next one's before they have landed.
    __syncthreads();
    if (tid == 0) {
      for (int i = 0; i < kStages; ++i)
        if (sh.holds[i] >= 0) mbar_wait_landed(&sh.full[i], sh.holds[i] / kStages & 1);
      atomicExch(status, kStatusTimeout);
    }
  }
}

// ---------------------------------------------------------------- host
struct Device {
  ScratchPool scratch;
  int* status = nullptr;
  long long next_wait_limit = 0;   // syfi_kv4_debug_wait_limit: applies to the next call, then clears itself
};
constexpr long long kWaitLimit = 1ll << 32;   // SM clocks without a finished tile (about two seconds)
std::mutex g_mu;
Device g_devices[64];

template <int D, int NT>
bool raise_decode() {
  return cudaFuncSetAttribute(kv4_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Decode4Shape<D, NT>::kSmem) == cudaSuccess;
}

constexpr size_t kTicketBytes = 4096;      // 1024 CTAs

bool take_scratch(AttentionArgs& a, Device& d, size_t partial, cudaStream_t st, int* rc) {
  ScratchBuffer* const s = d.scratch.get(st, kTicketBytes + partial, kTicketBytes, SYFI_KV4_ERR_CUDA, rc);
  if (!s) return false;
  a.tickets = static_cast<int*>(s->memory);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(s->memory) + kTicketBytes);
  return true;
}

template <int D, int NT>
int launch_decode(AttentionArgs a, Device& d, int sms, long long wait_limit, cudaStream_t st) {
  using Shape = Decode4Shape<D, NT>;
  const int ctas = sms * Shape::kBlocks;
  int rc = SYFI_KV4_OK;
  if (!take_scratch(a, d, 2ull * ctas * Shape::kRows * (D + 4) * sizeof(float), st, &rc)) return rc;
  return launch_dependent(kv4_decode_kernel<D, NT>, dim3(ctas), dim3(Shape::kThreads), Shape::kSmem, st, a, d.status, wait_limit) == cudaSuccess
             ? SYFI_KV4_OK : kv_fail(SYFI_KV4_ERR_CUDA, "attention kernel launch failed");
}

}  // namespace

}  // namespace syfi

using namespace syfi;

extern "C" int syfi_kv4_attention(const void* q, int64_t q_stride, const void* cache, int64_t num_pages, int64_t page_stride,
                                  const int32_t* block_table, int32_t max_pages, const int32_t* seq_lens,
                                  const int32_t* q_starts, int32_t batch, int64_t tokens, int32_t q_heads, int32_t kv_heads,
                                  int32_t head_dim, double scale, int32_t window, void* out, int64_t out_stride,
                                  void* stream) {
  if (const char* wrong = kv4_cache_error(cache, num_pages, page_stride, kv_heads, head_dim)) return kv_fail(SYFI_KV4_ERR_INVALID, wrong);
  if (q_heads < 1 || q_heads > 4096 || q_heads % kv_heads != 0) return kv_fail(SYFI_KV4_ERR_INVALID, "q_heads must be a multiple of kv_heads");
  if (batch < 0 || batch > (1 << 16)) return kv_fail(SYFI_KV4_ERR_INVALID, "batch out of range");
  if (tokens < 0 || tokens > 0x3fffffffll / q_heads) return kv_fail(SYFI_KV4_ERR_INVALID, "tokens out of range");
  if (max_pages < 1 || max_pages > (1 << 20)) return kv_fail(SYFI_KV4_ERR_INVALID, "max_pages (block table width) out of range");
  if (window < 0) return kv_fail(SYFI_KV4_ERR_INVALID, "window must not be negative");
  if (!(scale > -1e30 && scale < 1e30)) return kv_fail(SYFI_KV4_ERR_INVALID, "scale is not a finite float");
  if (batch == 0 || tokens == 0) return SYFI_KV4_OK;
  if (!kv_aligned(q) || !kv_aligned(out) || !kv_table_aligned(block_table) || !kv_table_aligned(seq_lens) || !kv_table_aligned(q_starts))
    return kv_fail(SYFI_KV4_ERR_INVALID, "a tensor argument is null or not aligned (16 bytes, int32 tables 4)");
  const int64_t width = static_cast<int64_t>(q_heads) * head_dim;
  if (!kv_stride_ok(q_stride, width) || !kv_stride_ok(out_stride, width))
    return kv_fail(SYFI_KV4_ERR_INVALID, "a token stride is smaller than the token's heads or no multiple of 8");
  const int sms = kv_device_sms();
  if (!sms) return SYFI_KV4_ERR_CUDA;
  AttentionArgs a = {};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.cache = {static_cast<uint8_t*>(const_cast<void*>(cache)), page_stride, static_cast<int>(num_pages), 2, kv_heads};
  a.batch = {block_table, seq_lens, q_starts, batch, max_pages, static_cast<int>(tokens)};
  a.group = q_heads / kv_heads;
  a.window = window < max_pages * kKvPage ? window : 0;      // (one as wide as any sequence is none; position - window stays in 32 bits)
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(g_mu);
  Device& d = g_devices[dev];
  if (!d.status) {
    if (!raise_decode<128, 1>() || !raise_decode<128, 2>() || !raise_decode<64, 1>() || !raise_decode<64, 2>() ||
        kv4_chunk_set_attributes() != cudaSuccess)
      return kv_fail(SYFI_KV4_ERR_CUDA, "cannot raise the shared-memory limit of the attention kernels");
    RelaxedCapture relaxed;
    int* fresh = nullptr;
    if (cudaMalloc(&fresh, 16) != cudaSuccess) return kv_fail(SYFI_KV4_ERR_CUDA, "out of device memory");
    if (!zero_now(fresh, 16)) {
      cudaFree(fresh);
      return kv_fail(SYFI_KV4_ERR_CUDA, "cannot clear the status word");
    }
    d.status = fresh;
  }
  const long long wait_limit = d.next_wait_limit > 0 ? d.next_wait_limit : kWaitLimit;
  d.next_wait_limit = 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Rows per sequence and key head, on average (the lengths themselves are on the device).  The decoding kernel reads a sequence's pages for
  // every 8 or 16 of them, the chunk kernel for every 256, but a tile costs it as much for 8 rows as for 256.  32 sequences of 16384 positions,
  // 8 key heads, us by rows:
  //                      4    8   12   16   24   32
  //   decoding, 8 rows  141  141  258  258  373  489
  //   decoding, 16           142  202  202  370  372
  //   chunks            494  495  495  495  498  499
  // One sequence of 65536: 38, 40, 51, 52, 64, 78 - 53, 53, 68, 71 from 12 rows - 111 to 125.  Heads of 64, with the kernel that is taken: 104 (4 and
  // 8 rows), 147 (12, 16), 262 (24), 265 (32), 396 (from 33 on); one sequence 36, 37, 44, 43, 55, 56 and 73.
  // The average is of all rows of q, those of no sequence among them.  It is far from right where few sequences of many rows meet many of few: 60
  // sequences of one token beside 400 tokens behind 60000 positions go to decoding and take 1948 us, in two calls 501; 64 sequences of 16384
  // positions beside a prompt of 2048 tokens go to the chunk kernel, 1093 and 347.
  const int64_t rows = (tokens * a.group + batch - 1) / batch;
  if (rows > 32) {
    int rc = SYFI_KV4_OK;
    if (!take_scratch(a, d, kv4_chunk_partial_bytes(head_dim, sms), st, &rc)) return rc;
    return launch_kv4_chunk(a, head_dim, sms, d.status, wait_limit, st) == cudaSuccess ? SYFI_KV4_OK : kv_fail(SYFI_KV4_ERR_CUDA, "attention kernel launch failed");
  }
  if (head_dim == 128) return rows <= 8 ? launch_decode<128, 1>(a, d, sms, wait_limit, st) : launch_decode<128, 2>(a, d, sms, wait_limit, st);
  return rows <= 8 ? launch_decode<64, 1>(a, d, sms, wait_limit, st) : launch_decode<64, 2>(a, d, sms, wait_limit, st);
}

// Test hook for the bounded waits, no part of the interface: a CTA of the next attention call's kernel on the current device may
// go without finishing a tile for this many SM clocks (0: the normal limit).
extern "C" int syfi_kv4_debug_wait_limit(int64_t clocks) {
  if (clocks < 0) return kv_fail(SYFI_KV4_ERR_INVALID, "a wait limit must not be negative");
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return kv_fail(SYFI_KV4_ERR_CUDA, "no current CUDA device");
  std::lock_guard<std::mutex> lock(g_mu);
  g_devices[dev].next_wait_limit = clocks;
  return SYFI_KV4_OK;
}

extern "C" int syfi_kv4_check(void* stream) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return kv_fail(SYFI_KV4_ERR_CUDA, "no current CUDA device");
  if (cudaStreamSynchronize(static_cast<cudaStream_t>(stream)) != cudaSuccess) return kv_fail(SYFI_KV4_ERR_CUDA, "stream synchronisation failed");
  std::lock_guard<std::mutex> lock(g_mu);
  Device& d = g_devices[dev];
  if (!d.status) return SYFI_KV4_OK;
  int status = 0;
  if (cudaMemcpy(&status, d.status, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) return kv_fail(SYFI_KV4_ERR_CUDA, "cannot read the status word");
  if (status != 0) {
    cudaMemset(d.status, 0, sizeof(int));
    char msg[128];
    snprintf(msg, sizeof(msg), "a kernel reported status %d (401: a bounded wait of the attention ran out; its rows are NaN)", status);
    return kv_fail(SYFI_KV4_ERR_DEVICE, msg);
  }
  return SYFI_KV4_OK;
}
