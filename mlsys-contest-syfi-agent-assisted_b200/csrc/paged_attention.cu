// Attention of new tokens over the quantised paged KV cache (include/syfi_kv.h).
//
//   x_j = scale * kscale_j * sum_d q_d k_jd,   out_d = sum_j exp(x_j) vscale_j v_jd / sum_j exp(x_j)   over the visible positions j
// in one pass over the cache.  With x in units of log2 and references m (of the sum l) and n (of the sum o) that follow the largest
// terms,   l = sum 2^(x_j - m),   o_d = sum 2^(x_j + log2 vscale_j - n) v_jd,   out_d = o_d 2^(n - m) / l :
// the values' scales go into the weights, so the products are made with the cache's e4m3 bytes as they are, which f16 holds exactly.
#include <cstdio>
#include <mutex>

#include "attention_common.cuh"
#include "stream_scratch.h"

namespace syfi {

namespace {

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float lg2(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The transpose of an 8 x 8 matrix of f16: lane 4 i + j has elements (i, 2 j) and (i, 2 j + 1) before, (2 j, i) and (2 j + 1, i) after.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// ---------------------------------------------------------------- few rows per sequence and key head: decoding
// A CTA walks its piece of the pages through a ring of stages filled by cp.async.  Four warps share a page, 16 positions each, for
// 8 NT rows; mma.sync m16n8k16 in f16, whose big operand the lanes make from the bytes in registers, so that a row tile is as narrow
// as an MMA allows:
//   scores:  positions (M) x rows (N) = K Q^T.  A lane's K operand is 16 bytes of two positions; the MMAs' k index permutes the dimensions,
//            alike in q.
//   values:  dimensions (M) x rows (N) = V^T P^T.  A lane's V operand pairs the bytes of two positions (prmt), its 16 dimensions are the m
//            indices of eight MMAs; the weights come from the scores' layout by an 8 x 8 transpose (movmatrix).
// Which position an index of the scores stands for is chosen so that both reads of the swizzled rows are free of bank conflicts: even i
// is position i, odd i is position (i - 1) ^ 5.
// What bounds it is the cache's bytes, so what counts is loads in flight and few instructions per page: 32 sequences of 65536 positions,
// 4 key heads of 128, 8 rows each: 347 us, 6.4 TB/s back to back, 374 to 403 us with other memory touched in between.  Short or few sequences: the chain of planning, a page's latency, and the join of
// parts (one sequence of 700 positions 13 us).
// What a unit costs besides its pages, in pages.  With 0, 1, 2, 4 (us, a flushed L2): 24 sequences of 300 .. 30000 positions, 8 rows 95, 94, 87,
// 87; 128 of 100 .. 3000 115, 91, 84, 81; 128 of 300 57, 55, 55, 55; 32 of 65536 360, 362, 362, 361.
constexpr int kDecodeExtra = 1;
constexpr float kFarBehind = 1.2676506e30f;   // 2^100 between the references of the two sums: the values' follows

template <int D, int NT>
struct DecodeShape {
  static constexpr int kRows = 8 * NT;
  static constexpr int kThreads = 128;
  static constexpr int kBlocks = NT == 1 ? 3 : 2;          // per SM
  static constexpr int kStages = D == 128 ? (NT == 1 ? 3 : 5) : (NT == 1 ? 5 : 9);
  static constexpr int kBlockBytes = kKvPage * D;
  static constexpr int kStageBytes = 2 * kBlockBytes + 2 * kKvPage * 4;
  static constexpr int kMerge = 2 * 8 * NT * D;                         // floats
  static constexpr int kSmem = kStages * kStageBytes + kMerge * 4;
};

template <int D, int NT>
__global__ void __launch_bounds__(DecodeShape<D, NT>::kThreads, DecodeShape<D, NT>::kBlocks) attention_decode_kernel(const __grid_constant__ AttentionArgs a) {
  using Shape = DecodeShape<D, NT>;
  constexpr int kRows = Shape::kRows, kStages = Shape::kStages, kSteps = D / 16, kMmas = D / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ PlanShared s_plan;
  __shared__ int s_there[kStages];
  __shared__ float4 s_stat[4][8 * NT];
  float* const s_merge = reinterpret_cast<float*>(smem + kStages * Shape::kStageBytes);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, c = lane % 4;

  pdl_wait();
  pdl_trigger();
  const Plan<kKvPage, kRows, kDecodeExtra> plan = {a.batch, a.cache.heads, a.group, a.window};
  const long long total = plan.total(s_plan);
  const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
  if (static_cast<int>(blockIdx.x) >= ctas) return;
  const long long w0 = piece_start(total, ctas, blockIdx.x), w1 = piece_start(total, ctas, blockIdx.x + 1);
  plan.locate(s_plan, w0);

  Cursor<kKvPage, kRows, kDecodeExtra> load, use;
  load.start(plan, s_plan, static_cast<int>(w1 - w0));
  if (load.left <= 0) return;
  use = load;
  int stage_in = 0, stage_out = 0;           // of the page to ask for, of the page to work on
  auto entry_of = [&](const Cursor<kKvPage, kRows, kDecodeExtra>& at) {
    return __ldg(a.batch.block_table + static_cast<long long>(at.b) * a.batch.max_pages + at.span.first + at.tile);
  };
  const int to_values = a.cache.heads * (kKvPage * (D + 4));
  int entry = entry_of(load);                // of the page to ask for next: read one page ahead
  auto ask = [&]() {
    if (load.left > 0) {
      const int stage = stage_in;
      stage_in = stage_in + 1 == kStages ? 0 : stage_in + 1;
      const bool there = entry >= 0 && entry < a.cache.num_pages;
      if (there) {
        // a thread's chunks lie kThreads apart, a multiple of eight rows: they differ by constants
        constexpr int kChunks = Shape::kBlockBytes / 16, kEach = (kChunks + Shape::kThreads - 1) / Shape::kThreads;
        static_assert(Shape::kThreads % (8 * (D / 16)) == 0, "the swizzle repeats every eight rows");
        const uint32_t base = smem_u32(smem) + stage * Shape::kStageBytes, dst = base + swizzled<D>(tid / (D / 16), tid % (D / 16));
        const uint8_t* const k_block = kv_block<D>(a.cache, entry, 0, load.head);
        const uint8_t* const v_block = k_block + to_values;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          if (kChunks % Shape::kThreads == 0 || tid + i * Shape::kThreads < kChunks) {
            cp_async16(dst + i * Shape::kThreads * 16, k_block + (tid + i * Shape::kThreads) * 16);
            cp_async16(dst + Shape::kBlockBytes + i * Shape::kThreads * 16, v_block + (tid + i * Shape::kThreads) * 16);
          }
        }
        if (tid < 32) cp_async16(base + 2 * Shape::kBlockBytes + tid * 16, (tid < 16 ? k_block : v_block) + Shape::kBlockBytes + tid % 16 * 16);
      }
      if (tid == 0) s_there[stage] = there;
      load.advance(plan, 1);
      if (load.left > 0) entry = entry_of(load);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) ask();

  // This lane's positions of a page: t0 and t0 + 8; its rows of the scores: 8 t + 2 c and 8 t + 2 c + 1.
  const int t0 = warp * 16 + ((g & 1) ? (g - 1) ^ 5 : g);
  uint32_t qb[NT][kSteps][2];
  // Of each row: what a score is worth; the reference of this lane's sum, and the sum; the reference of the values' sum, and 2^(m - n + 7).
  float unit[NT][2], m[NT][2], l[NT][2], n[NT][2], up[NT][2], o[NT][kMmas][4];
  int low[NT][2], high[NT][2];               // positions that the rows see
  int all_low = 0, all_high = 0, any_low = 0, any_high = 0;   // positions that all / any of the unit's rows see
  bool fresh = true;
  int begun = use.tile;                      // the segment's first tile

  while (use.left > 0) {
    cp_async_wait<kStages - 2>();
    __syncthreads();
    ask();
    if (fresh) {
      fresh = false;
      begun = use.tile;
      const int rows = use.rows(a.group), base = use.s.length - use.s.count, r0 = use.rt * kRows;
      const int first = base + r0 / a.group, last = base + (r0 + rows - 1) / a.group;
      all_low = a.window > 0 ? max(last - a.window + 1, 0) : 0;
      any_low = a.window > 0 ? max(first - a.window + 1, 0) : 0;
      all_high = first;
      any_high = last;
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
          raw[step] = real ? __ldg(reinterpret_cast<const uint2*>(from + 16 * (c + 4 * (step / 4)) + 4 * (step % 4))) : make_uint2(0u, 0u);
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
    }

    const int stage = stage_out;
    stage_out = stage_out + 1 == kStages ? 0 : stage_out + 1;
    uint8_t* const keys = smem + stage * Shape::kStageBytes;
    uint8_t* const values = keys + Shape::kBlockBytes;
    float* const k_scale = reinterpret_cast<float*>(keys + 2 * Shape::kBlockBytes);
    float* const v_scale = k_scale + kKvPage;
    const int position0 = (use.span.first + use.tile) * kKvPage;
    const bool plain = position0 >= all_low && position0 + kKvPage - 1 <= all_high;    // every row sees every position of the page
    if (s_there[stage]) {
      if (!plain) {
        // What a row does not see must not reach its sums, and zero times NaN is NaN: positions that no row sees lose their bytes, and
        // where some rows see a value that is not finite, the NaN goes by way of its score to those rows alone.
        for (int t = tid / 2; t < kKvPage; t += Shape::kThreads / 2) {
          const int half = tid % 2, position = position0 + t;
          const bool unseen = position < any_low || position > any_high;
          bool bad = false;
          uint4* const chunk0 = reinterpret_cast<uint4*>(values);
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const uint4 w = chunk0[swizzled<D>(t, half * (D / 32) + i) / 16];
            const uint32_t over = ((w.x & 0x7f7f7f7fu) + 0x01010101u) | ((w.y & 0x7f7f7f7fu) + 0x01010101u) |
                                  ((w.z & 0x7f7f7f7fu) + 0x01010101u) | ((w.w & 0x7f7f7f7fu) + 0x01010101u);
            bad |= (over & 0x80808080u) != 0u;
          }
          bad = __shfl_xor_sync(0xffffffffu, static_cast<int>(bad), 1) | static_cast<int>(bad);
          bad |= !(fabsf(v_scale[t]) <= 3.402823466e38f);
          __syncwarp();
          if (bad || unseen) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) chunk0[swizzled<D>(t, half * (D / 32) + i) / 16] = make_uint4(0u, 0u, 0u, 0u);
            if (half == 0) {
              v_scale[t] = 1.0f;
              if (bad) k_scale[t] = __int_as_float(0x7fffffff);
            }
          }
        }
        __syncthreads();
      }
      float x[NT][4];
      {
        float even[NT][4], odd[NT][4];       // two chains of MMAs
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) even[t][e] = odd[t][e] = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
          const uint4 p = *reinterpret_cast<const uint4*>(keys + swizzled<D>(t0, c + 4 * j)), r = *reinterpret_cast<const uint4*>(keys + swizzled<D>(t0 + 8, c + 4 * j));
          const uint32_t w[4] = {p.x, p.y, p.z, p.w}, v[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t ka[4] = {e4m3x2_to_half2(w[i]), e4m3x2_to_half2(v[i]), e4m3x2_to_half2(w[i] >> 16), e4m3x2_to_half2(v[i] >> 16)};
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_f16(i & 1 ? odd[t] : even[t], ka, qb[t][4 * j + i][0], qb[t][4 * j + i][1]);
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[t][e] = even[t][e] + odd[t][e];
      }
      const float ks[2] = {k_scale[t0], k_scale[t0 + 8]}, vs[2] = {v_scale[t0], v_scale[t0 + 8]};
      bool grown = false, late = false;
      // element e: position t0 + 8 (e / 2), row 2 c + e % 2
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[t][e] *= ks[e / 2] * unit[t][e % 2];
      if (!plain) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int position = position0 + t0 + 8 * (e / 2);
            if (position < low[t][e % 2] || position > high[t][e % 2]) x[t][e] = -INFINITY;
          }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) grown |= fmaxf(x[t][i], x[t][2 + i]) > m[t][i] + kSumGrowth;
      if (__any_sync(0xffffffffu, grown)) {
        // a row's sum in this lane follows its scores once they are 2^16 above the reference; the lanes meet at the unit's end
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float top = fmaxf(x[t][i], x[t][2 + i]);
            if (top > m[t][i] + kSumGrowth) {
              l[t][i] *= ex2(m[t][i] - top);
              m[t][i] = top;
              up[t][i] = n[t][i] == -INFINITY ? 0.0f : ex2(top - n[t][i] + kHeadroom);
              late |= up[t][i] > kFarBehind;
            }
          }
      }
      float p[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float m_ref[2] = {finite_or_zero(m[t][0]), finite_or_zero(m[t][1])};
#pragma unroll
        for (int e = 0; e < 4; ++e) p[t][e] = ex2(x[t][e] - m_ref[e % 2]);
        l[t][0] += p[t][0] + p[t][2];
        l[t][1] += p[t][1] + p[t][3];
#pragma unroll
        for (int e = 0; e < 4; ++e) p[t][e] *= vs[e / 2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float top = fmaxf(p[t][i], p[t][2 + i]);
          late |= top * up[t][i] > 32768.0f || (up[t][i] == 0.0f && top > 0.0f);
        }
      }
      if (__any_sync(0xffffffffu, late)) {
        // the reference of the values' sum follows, in all lanes of a row alike
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float fade[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = m[t][i] + fmaxf(lg2(fmaxf(p[t][i], p[t][2 + i])), -90.0f);      // (never further behind: a value may be zero)
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            fade[i] = 1.0f;
            if (top > n[t][i] + kGrowth) {
              fade[i] = ex2(n[t][i] - top);
              n[t][i] = top;
            }
            up[t][i] = n[t][i] == -INFINITY || m[t][i] == -INFINITY ? 0.0f : ex2(m[t][i] - n[t][i] + kHeadroom);
          }
#pragma unroll
          for (int j = 0; j < kMmas; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][j][e] *= fade[e % 2];
        }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) pb[t][u] = transposed(pack_half2(p[t][2 * u] * up[t][0], p[t][2 * u + 1] * up[t][1]));
      uint32_t even[2][D / 32], odd[2][D / 32];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int v0 = warp * 16 + 8 * u + 2 * c, v1 = warp * 16 + 8 * u + ((2 * c) ^ 5);
        if constexpr (D == 128) {
          const uint4 w = *reinterpret_cast<const uint4*>(values + swizzled<D>(v0, g)), r = *reinterpret_cast<const uint4*>(values + swizzled<D>(v1, g));
          even[u][0] = w.x; even[u][1] = w.y; even[u][2] = w.z; even[u][3] = w.w;
          odd[u][0] = r.x; odd[u][1] = r.y; odd[u][2] = r.z; odd[u][3] = r.w;
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(values + swizzled<D>(v0, g / 2) + (g & 1) * 8), r = *reinterpret_cast<const uint2*>(values + swizzled<D>(v1, g / 2) + (g & 1) * 8);
          even[u][0] = w.x; even[u][1] = w.y;
          odd[u][0] = r.x; odd[u][1] = r.y;
        }
      }
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // dimensions 4 w + 2 h and 4 w + 2 h + 1 of this lane's D / 8
          const uint32_t b0 = __byte_perm(even[0][w], odd[0][w], h ? 0x7362 : 0x5140), b1 = __byte_perm(even[1][w], odd[1][w], h ? 0x7362 : 0x5140);
          const uint32_t va[4] = {e4m3x2_to_half2(b0), e4m3x2_to_half2(b0 >> 16), e4m3x2_to_half2(b1), e4m3x2_to_half2(b1 >> 16)};
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_f16(o[t][2 * w + h], va, pb[t][0], pb[t][1]);
        }
      }
    }

    const bool unit_ends = use.tile + 1 == use.span.tiles;
    if (unit_ends || use.left == 1) {
      // ---- the segment's end: lanes, then the four warps of a row group, then the unit's other pieces
      const int rows = use.rows(a.group);
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
          if (g == 0) s_stat[warp][8 * t + 2 * c + i] = make_float4(top, sum, n[t][i], 0.0f);
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
            m_all = fmaxf(m_all, s_stat[w][8 * t + 2 * c + i].x);
            n_all = fmaxf(n_all, s_stat[w][8 * t + 2 * c + i].z);
          }
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float4 st = s_stat[w][8 * t + 2 * c + i];
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
      const bool whole = begun == 0 && unit_ends;
      const long long unit_start = w1 - use.left - use.tile;      // the place of its first page
      if (warp == 0) {
        const float* other = s_merge + 8 * NT * D + lane;
        const int slot = 2 * static_cast<int>(blockIdx.x) + (w0 >= unit_start ? 0 : 1);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = t * 8 + 2 * c + i, r = use.rt * kRows + row;
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
      // (what the next segment sets anyway: not kept in registers across the join, whose own made the loop above spill)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int step = 0; step < kSteps; ++step) qb[t][step][0] = qb[t][step][1] = 0u;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          unit[t][i] = m[t][i] = l[t][i] = n[t][i] = up[t][i] = 0.0f;
          low[t][i] = high[t][i] = 0;
        }
#pragma unroll
        for (int j = 0; j < kMmas; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[t][j][e] = 0.0f;
      }
      if (!whole) {
        const Parts parts(total, ctas, unit_start, use.span.tiles);
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
          join_parts<D, kRows>(a, use.s.first, use.rt * kRows, use.head, rows, ctas, parts, warp, 4);
        }
      }
      fresh = true;
    }
    use.advance(plan, 1);
  }
}

// ---------------------------------------------------------------- host
struct Device {
  ScratchPool scratch;
  int* status = nullptr;
  long long next_wait_limit = 0;   // syfi_kv_debug_wait_limit: applies to the next call, then clears itself
};
constexpr long long kWaitLimit = 1ll << 32;   // SM clocks without a finished tile (about two seconds)
std::mutex g_mu;
Device g_devices[64];

template <int D, int NT>
bool raise_decode() {
  return cudaFuncSetAttribute(attention_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodeShape<D, NT>::kSmem) == cudaSuccess;
}

constexpr size_t kTicketBytes = 4096;      // 1024 CTAs

bool take_scratch(AttentionArgs& a, Device& d, size_t partial, cudaStream_t st, int* rc) {
  ScratchBuffer* const s = d.scratch.get(st, kTicketBytes + partial, kTicketBytes, SYFI_KV_ERR_CUDA, rc);
  if (!s) return false;
  a.tickets = static_cast<int*>(s->memory);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(s->memory) + kTicketBytes);
  return true;
}

template <int D, int NT>
int launch_decode(AttentionArgs a, Device& d, int sms, cudaStream_t st) {
  using Shape = DecodeShape<D, NT>;
  const int ctas = sms * Shape::kBlocks;
  int rc = SYFI_KV_OK;
  if (!take_scratch(a, d, 2ull * ctas * Shape::kRows * (D + 4) * sizeof(float), st, &rc)) return rc;
  return launch_dependent(attention_decode_kernel<D, NT>, dim3(ctas), dim3(Shape::kThreads), Shape::kSmem, st, a) == cudaSuccess
             ? SYFI_KV_OK : kv_fail(SYFI_KV_ERR_CUDA, "attention kernel launch failed");
}

}  // namespace

}  // namespace syfi

using namespace syfi;

extern "C" int syfi_paged_attention(const void* q, int64_t q_stride, const void* cache, int64_t num_pages, int64_t page_stride,
                                    const int32_t* block_table, int32_t max_pages, const int32_t* seq_lens,
                                    const int32_t* q_starts, int32_t batch, int64_t tokens, int32_t q_heads, int32_t kv_heads,
                                    int32_t head_dim, double scale, int32_t window, void* out, int64_t out_stride,
                                    void* stream) {
  if (const char* wrong = kv_cache_error(cache, num_pages, page_stride, 2, kv_heads, head_dim)) return kv_fail(SYFI_KV_ERR_INVALID, wrong);
  if (q_heads < 1 || q_heads > 4096 || q_heads % kv_heads != 0) return kv_fail(SYFI_KV_ERR_INVALID, "q_heads must be a multiple of kv_heads");
  if (batch < 0 || batch > (1 << 16)) return kv_fail(SYFI_KV_ERR_INVALID, "batch out of range");
  if (tokens < 0 || tokens > 0x3fffffffll / q_heads) return kv_fail(SYFI_KV_ERR_INVALID, "tokens out of range");
  if (max_pages < 1 || max_pages > (1 << 20)) return kv_fail(SYFI_KV_ERR_INVALID, "max_pages (block table width) out of range");
  if (window < 0) return kv_fail(SYFI_KV_ERR_INVALID, "window must not be negative");
  if (!(scale > -1e30 && scale < 1e30)) return kv_fail(SYFI_KV_ERR_INVALID, "scale is not a finite float");
  if (batch == 0 || tokens == 0) return SYFI_KV_OK;
  if (!kv_aligned(q) || !kv_aligned(out) || !kv_table_aligned(block_table) || !kv_table_aligned(seq_lens) || !kv_table_aligned(q_starts))
    return kv_fail(SYFI_KV_ERR_INVALID, "a tensor argument is null or not aligned (16 bytes, int32 tables 4)");
  const int64_t width = static_cast<int64_t>(q_heads) * head_dim;
  if (!kv_stride_ok(q_stride, width) || !kv_stride_ok(out_stride, width))
    return kv_fail(SYFI_KV_ERR_INVALID, "a token stride is smaller than the token's heads or no multiple of 8");
  const int sms = kv_device_sms();
  if (!sms) return SYFI_KV_ERR_CUDA;
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
        chunk_set_attributes() != cudaSuccess)
      return kv_fail(SYFI_KV_ERR_CUDA, "cannot raise the shared-memory limit of the attention kernels");
    RelaxedCapture relaxed;
    if (cudaMalloc(&d.status, 16) != cudaSuccess || !zero_now(d.status, 16)) return kv_fail(SYFI_KV_ERR_CUDA, "out of device memory");
  }
  const long long wait_limit = d.next_wait_limit > 0 ? d.next_wait_limit : kWaitLimit;
  d.next_wait_limit = 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Rows per sequence and key head, on average (the lengths themselves are on the device): row tiles of 8 or 16, beyond that the tensor
  // memory kernel's.  24 sequences of 300 .. 30000 positions, 8 key heads of 128, us for 8 | 16 | 32 rows each: tiles of 8 79 | 134 | 249,
  // tiles of 16 121 | 129 | 259, the tensor memory kernel 141 | 143 | 145.  Unequal rows, a chunk of 512 tokens behind 4000 positions beside
  // 24 | 100 | 256 | 500 sequences of 2000 with one token, 4 rows a token: row tiles 293 | 381 | 592 | 903, the tensor memory kernel
  // 117 | 271 | 536 | 1079 (each half alone in its own kernel: the chunk 70, 256 sequences 257).
  const int64_t rows = (tokens * a.group + batch - 1) / batch;
  if (rows > 16) {
    int rc = SYFI_KV_OK;
    if (!take_scratch(a, d, chunk_partial_bytes(head_dim, sms), st, &rc)) return rc;
    return launch_chunk(a, head_dim, sms, d.status, wait_limit, st) == cudaSuccess ? SYFI_KV_OK : kv_fail(SYFI_KV_ERR_CUDA, "attention kernel launch failed");
  }
  if (head_dim == 128) return rows <= 8 ? launch_decode<128, 1>(a, d, sms, st) : launch_decode<128, 2>(a, d, sms, st);
  return rows <= 8 ? launch_decode<64, 1>(a, d, sms, st) : launch_decode<64, 2>(a, d, sms, st);
}

// Test hook for the bounded waits, no part of the interface: a CTA of the next attention call's kernel on the current device may
// go without finishing a tile for this many SM clocks (0: the normal limit).
extern "C" int syfi_kv_debug_wait_limit(int64_t clocks) {
  if (clocks < 0) return kv_fail(SYFI_KV_ERR_INVALID, "a wait limit must not be negative");
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return kv_fail(SYFI_KV_ERR_CUDA, "no current CUDA device");
  std::lock_guard<std::mutex> lock(g_mu);
  g_devices[dev].next_wait_limit = clocks;
  return SYFI_KV_OK;
}

extern "C" int syfi_kv_check(void* stream) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return kv_fail(SYFI_KV_ERR_CUDA, "no current CUDA device");
  if (cudaStreamSynchronize(static_cast<cudaStream_t>(stream)) != cudaSuccess) return kv_fail(SYFI_KV_ERR_CUDA, "stream synchronisation failed");
  std::lock_guard<std::mutex> lock(g_mu);
  Device& d = g_devices[dev];
  if (!d.status) return SYFI_KV_OK;
  int status = 0;
  if (cudaMemcpy(&status, d.status, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) return kv_fail(SYFI_KV_ERR_CUDA, "cannot read the status word");
  if (status != 0) {
    cudaMemset(d.status, 0, sizeof(int));
    char msg[128];
    snprintf(msg, sizeof(msg), "a kernel reported status %d (301: a bounded wait of the attention ran out; its rows are NaN)", status);
    return kv_fail(SYFI_KV_ERR_DEVICE, msg);
  }
  return SYFI_KV_OK;
}
