// Shared by the two attention kernels: their arguments, small device functions, and how a split unit's parts are added up.
#pragma once
#include "attention_plan.cuh"
#include "kv_internal.h"

namespace syfi {

struct AttentionArgs {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  long long q_stride, out_stride;
  KvCache cache;
  KvBatch batch;
  int group, window;
  float scale_log2;
  int* tickets;          // [CTAs] zero between calls
  float* partial;        // [2 * CTAs][rows][D] sums (the chunk kernel: [2 * CTAs][D / 4][rows][4]), then [2 * CTAs][rows] of (m, l, n, doubt)
};

// paged_attention_chunk.cu.  Bytes of `partial` that a launch on `ctas` CTAs needs, and the launch.
size_t chunk_partial_bytes(int head_dim, int ctas);
cudaError_t chunk_set_attributes();
cudaError_t launch_chunk(const AttentionArgs& a, int head_dim, int ctas, int* status, long long wait_limit, cudaStream_t st);

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t bytes) {   // the lower two
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(bytes)));
  return h;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.0f : m; }


constexpr float kHeadroom = 7.0f;     // weights are kept times 2^7 in f16 ...
constexpr float kGrowth = 8.0f;       // ... and may grow to 2^15 before their reference follows
constexpr float kSumGrowth = 16.0f;   // a sum of weights in f32 lets them grow further


template <int D>
__device__ __forceinline__ int swizzled(int row, int chunk) {   // byte offset of a row's 16-byte chunk
  return row * D + ((D == 128 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3)) << 4);
}

// The parts of a split unit whose tiles are the places [unit_start, unit_start + tiles) of the line: CTAs first .. last, of which all but
// perhaps the first have it at the start of their piece.
struct Parts {
  int first, last, first_slot;
  __device__ Parts(int f, int l, int s) : first(f), last(l), first_slot(s) {}
  __device__ Parts(long long total, int ctas, long long unit_start, int tiles)
      : first(piece_of(total, ctas, unit_start)), last(piece_of(total, ctas, unit_start + tiles - 1)),
        first_slot(2 * first + (piece_start(total, ctas, first) < unit_start)) {}
  __device__ int slot(int c) const { return c == first ? first_slot : 2 * c; }
};

// Adds up a split unit's parts: out = sum o_p 2^(n_p - n) 2^(n - m) / sum l_p 2^(m_p - m).  A warp has two rows at a time; its lanes
// read the statistics of 32 parts at once and come to their factors, then each lane has four dimensions and eight parts' loads under
// way.  One part after the other, a row of 55 parts (one sequence of 60000 positions) took 16 us of the call's 50.
template <int D, int ROWS>
__device__ __forceinline__ void join_parts(const AttentionArgs& a, int q_first, int unit_row0, int head, int rows, int ctas, const Parts& parts,
                                           int warp, int warps) {
  constexpr int kLanes = D / 4, kTogether = 32 / kLanes, kLoads = 8, kBatch = 2;
  const float4* const stats = reinterpret_cast<const float4*>(a.partial + 2ll * ctas * ROWS * D);
  const int lane = threadIdx.x % 32, d = lane % kLanes * 4, sub = lane / kLanes;
  for (int row0 = warp; row0 < rows; row0 += warps * kBatch) {
    float m[kBatch], n[kBatch], l[kBatch];
    float4 o[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      m[b] = n[b] = -INFINITY;
      l[b] = 0.0f;
      o[b] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    for (int base = parts.first; base <= parts.last; base += 32) {
      const int count = min(parts.last - base + 1, 32);
      float4 st[kBatch];
      float w[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        st[b] = make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
        if (lane < count && row0 + b * warps < rows) st[b] = __ldcg(stats + static_cast<long long>(parts.slot(base + lane)) * ROWS + row0 + b * warps);
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        float m_new = fmaxf(m[b], st[b].x), n_new = fmaxf(n[b], st[b].z);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) {
          m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, x));
          n_new = fmaxf(n_new, __shfl_xor_sync(0xffffffffu, n_new, x));
        }
        const float m_ref = finite_or_zero(m_new), n_ref = finite_or_zero(n_new), fade = ex2(n[b] - n_ref);
        float sum = st[b].y * ex2(st[b].x - m_ref);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        l[b] = l[b] * ex2(m[b] - m_ref) + sum;
        o[b] = make_float4(o[b].x * fade, o[b].y * fade, o[b].z * fade, o[b].w * fade);
        w[b] = ex2(st[b].z - n_ref);
        m[b] = m_new;
        n[b] = n_new;
      }
#pragma unroll 1
      for (int k0 = 0; k0 < count; k0 += kLoads * kTogether) {
        float4 p[kBatch][kLoads];
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            const int k = k0 + i * kTogether + sub;
            p[b][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (k < count && row0 + b * warps < rows)
              p[b][i] = __ldcg(reinterpret_cast<const float4*>(a.partial + (static_cast<long long>(parts.slot(base + k)) * ROWS + row0 + b * warps) * D + d));
          }
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            const float f = __shfl_sync(0xffffffffu, w[b], k0 + i * kTogether + sub);
            o[b] = make_float4(o[b].x + p[b][i].x * f, o[b].y + p[b][i].y * f, o[b].z + p[b][i].z * f, o[b].w + p[b][i].w * f);
          }
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if constexpr (kTogether == 2) {
        o[b].x += __shfl_xor_sync(0xffffffffu, o[b].x, 16);
        o[b].y += __shfl_xor_sync(0xffffffffu, o[b].y, 16);
        o[b].z += __shfl_xor_sync(0xffffffffu, o[b].z, 16);
        o[b].w += __shfl_xor_sync(0xffffffffu, o[b].w, 16);
      }
      const int row = row0 + b * warps, r = unit_row0 + row;
      if (row >= rows || sub != 0) continue;
      const float f = l[b] == 0.0f || n[b] == -INFINITY ? 0.0f : ex2(n[b] - finite_or_zero(m[b]) - kHeadroom) / l[b];
      __nv_bfloat16* to = a.out + (q_first + r / a.group) * a.out_stride + (head * a.group + r % a.group) * D + d;
      const __nv_bfloat162 lo = __floats2bfloat162_rn(o[b].x * f, o[b].y * f), hi = __floats2bfloat162_rn(o[b].z * f, o[b].w * f);
      *reinterpret_cast<uint2*>(to) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  }
}

}  // namespace syfi
