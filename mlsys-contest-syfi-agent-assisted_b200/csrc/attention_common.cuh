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
  float* partial;        // [2 * CTAs][rows][D] sums, then [2 * CTAs][rows] of (m, l, n, redo)
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


template <int D>
__device__ __forceinline__ int swizzled(int row, int chunk) {   // byte offset of a row's 16-byte chunk
  return row * D + ((D == 128 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3)) << 4);
}

// Adds up a split unit's parts: out = sum o_p 2^(n_p - n) 2^(n - m) / sum l_p 2^(m_p - m).
template <int D, int ROWS>
__device__ __forceinline__ void join_parts(const AttentionArgs& a, const KvSequence& s, int rt, int head, int rows, long long total, int ctas, int first, int last,
                           long long unit_start, int thread, int threads) {
  const float4* stats = reinterpret_cast<const float4*>(a.partial + 2ll * ctas * ROWS * D);
  for (int i = thread; i < rows * (D / 4); i += threads) {
    const int row = i / (D / 4), d = (i % (D / 4)) * 4;
    auto slot = [&](int c) { return 2 * c + (piece_start(total, ctas, c) >= unit_start ? 0 : 1); };
    float m = -INFINITY, n = -INFINITY;
    for (int c = first; c <= last; ++c) {
      const float4 st = __ldcg(stats + static_cast<long long>(slot(c)) * ROWS + row);
      m = fmaxf(m, st.x);
      n = fmaxf(n, st.z);
    }
    const float m_ref = finite_or_zero(m), n_ref = finite_or_zero(n);
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int c = first; c <= last; ++c) {
      const long long at = static_cast<long long>(slot(c)) * ROWS + row;
      const float4 st = __ldcg(stats + at);
      const float4 part = __ldcg(reinterpret_cast<const float4*>(a.partial + at * D + d));
      l += st.y * ex2(st.x - m_ref);
      const float f = ex2(st.z - n_ref);
      o.x = fmaf(part.x, f, o.x);
      o.y = fmaf(part.y, f, o.y);
      o.z = fmaf(part.z, f, o.z);
      o.w = fmaf(part.w, f, o.w);
    }
    const float f = l == 0.0f ? 0.0f : ex2(n_ref - m_ref - kHeadroom) / l;
    const int r = rt * ROWS + row;
    __nv_bfloat16* to = a.out + (s.first + r / a.group) * a.out_stride + (head * a.group + r % a.group) * D + d;
    const __nv_bfloat162 lo = __floats2bfloat162_rn(o.x * f, o.y * f), hi = __floats2bfloat162_rn(o.z * f, o.w * f);
    *reinterpret_cast<uint2*>(to) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  }
}

}  // namespace syfi
