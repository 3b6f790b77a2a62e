// Shared by the translation units of the paged KV cache in 4 bits: the cache's layout (include/syfi_kv4.h) and its checks.
#pragma once
#include "../../include/syfi_kv4.h"
#include "attention_common.cuh"
#include "kv_internal.h"

namespace syfi {

constexpr int kKv4Group = 16;                 // dimensions that share a group scale
constexpr int kKv4Plane = kKvPage * 32;       // bytes of a page's codes of 64 dimensions

// Offsets inside a block: a page's tokens of one kind (0 keys, 1 values) and head.
template <int D>
struct Kv4Block {
  static constexpr int kGroups = kKvPage * (D / 2);                   // [token][D / 16]
  static constexpr int kScales = kGroups + kKvPage * (D / kKv4Group);  // [token]
  static constexpr int kBytes = kScales + kKvPage * 4;
};
template <int D>
__device__ __forceinline__ uint8_t* kv4_block(const KvCache& c, int page, int kind, int head) {
  return c.base + page * c.page_stride + static_cast<long long>(kind * c.heads + head) * Kv4Block<D>::kBytes;
}

// Byte K of a word holds two codes: as f16 values, the lower code's in the lower half.
template <int K>
__device__ __forceinline__ uint32_t e2m1x2_to_half2(uint32_t word) {
  static_assert(K >= 0 && K < 4, "a byte of the word");
  uint32_t h;
  if constexpr (K == 0) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(h) : "r"(word));
  if constexpr (K == 1) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(h) : "r"(word));
  if constexpr (K == 2) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, c;\n\t}" : "=r"(h) : "r"(word));
  if constexpr (K == 3) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, d;\n\t}" : "=r"(h) : "r"(word));
  return h;
}
// Eight values to the codes of a word, the first in its lowest bits: to nearest, to even between two, at most 6.
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float (&x)[8]) {
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w) : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return w;
}
__device__ __forceinline__ uint32_t hmul2_bits(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The cache's arguments as every entry point takes them; null when they are in order, else what is wrong.
inline const char* kv4_cache_error(const void* base, int64_t num_pages, int64_t page_stride, int32_t heads, int32_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return "head_dim must be 64 or 128";
  if (heads < 1 || heads > 1024) return "kv_heads out of range";
  if (num_pages < 1 || num_pages > (1ll << 24)) return "num_pages out of range";
  if (page_stride < 2ll * heads * kKvPage * (head_dim / 2 + head_dim / kKv4Group + 4) || page_stride % 16 != 0 || page_stride > (1ll << 36))
    return "page_stride is smaller than a page or no multiple of 16";
  if (!base || (reinterpret_cast<uintptr_t>(base) & 15u)) return "the cache is null or not 16-byte aligned";
  return nullptr;
}

}  // namespace syfi
