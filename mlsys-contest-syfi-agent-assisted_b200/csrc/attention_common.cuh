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
  float* partial;        // [2 * CTAs][rows][D] sums (the chunk kernel: [2 * CTAs][D / 4][rows][4]), then [2 * CTAs][rows] of (m, l, n, redo)
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

// Adds up a split unit's parts: out = sum o_p 2^(n_p - n) 2^(n - m) / sum l_p 2^(m_p - m).  A group of D / 4 threads has a row, four
// dimensions each, and BATCH rows at once, so that their loads are under way together.
template <int D, int ROWS, int BATCH>
__device__ __forceinline__ void join_parts(const AttentionArgs& a, int q_first, int unit_row0, int head, int rows, int ctas, const Parts& parts,
                                           int thread, int threads) {
  const float4* const stats = reinterpret_cast<const float4*>(a.partial + 2ll * ctas * ROWS * D);
  const int d = thread % (D / 4) * 4, groups = threads / (D / 4);
  for (int row0 = thread / (D / 4); row0 < rows; row0 += groups * BATCH) {
    float m[BATCH], n[BATCH], l[BATCH];
    float4 o[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      m[k] = n[k] = -INFINITY;
      l[k] = 0.0f;
      o[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll 2
    for (int c = parts.first; c <= parts.last; ++c) {
      const long long base = static_cast<long long>(parts.slot(c)) * ROWS;
      float4 st[BATCH], part[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const long long at = base + min(row0 + groups * k, rows - 1);
        st[k] = __ldcg(stats + at);
        part[k] = __ldcg(reinterpret_cast<const float4*>(a.partial + at * D + d));
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const float m_new = fmaxf(m[k], st[k].x), n_new = fmaxf(n[k], st[k].z), m_ref = finite_or_zero(m_new), n_ref = finite_or_zero(n_new);
        l[k] = l[k] * ex2(m[k] - m_ref) + st[k].y * ex2(st[k].x - m_ref);
        const float f = ex2(n[k] - n_ref), g = ex2(st[k].z - n_ref);
        o[k] = make_float4(o[k].x * f + part[k].x * g, o[k].y * f + part[k].y * g, o[k].z * f + part[k].z * g, o[k].w * f + part[k].w * g);
        m[k] = m_new;
        n[k] = n_new;
      }
    }
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int row = row0 + groups * k, r = unit_row0 + row;
      if (row >= rows) break;
      const float f = l[k] == 0.0f ? 0.0f : ex2(finite_or_zero(n[k]) - finite_or_zero(m[k]) - kHeadroom) / l[k];
      __nv_bfloat16* to = a.out + (q_first + r / a.group) * a.out_stride + (head * a.group + r % a.group) * D + d;
      const __nv_bfloat162 lo = __floats2bfloat162_rn(o[k].x * f, o[k].y * f), hi = __floats2bfloat162_rn(o[k].z * f, o[k].w * f);
      *reinterpret_cast<uint2*>(to) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  }
}

}  // namespace syfi
