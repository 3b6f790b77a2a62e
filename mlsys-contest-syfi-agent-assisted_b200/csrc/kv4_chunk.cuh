// What the two attention kernels over the 4-bit cache share besides its layout: the chunk kernel's launch, and the tcgen05 forms that only it uses.
#pragma once
#include "kv4_internal.h"

namespace syfi {

// kv4_attention_chunk.cu.  Bytes of `partial` that a launch on `ctas` CTAs needs, and the launch.
size_t kv4_chunk_partial_bytes(int head_dim, int ctas);
cudaError_t kv4_chunk_set_attributes();
cudaError_t launch_kv4_chunk(const AttentionArgs& a, int head_dim, int ctas, int* status, long long wait_limit, cudaStream_t st);

__device__ __forceinline__ float lg2(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint64_t f32x2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// Instruction descriptor: f32 accumulator, A and B f16, both K-major, M = 128, N = n.
__device__ __forceinline__ uint32_t umma_idesc_f16_m128(uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((128u >> 4) << 24); }
// D[tmem] (+)= A[smem] * B[smem]^T, f16 x f16 -> f32; descriptors given as their lower words and the upper word of both.
__device__ __forceinline__ void umma_f16_words(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %3};\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}"
      ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

}  // namespace syfi
