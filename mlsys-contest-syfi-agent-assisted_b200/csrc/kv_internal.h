// Shared by the translation units of the quantised paged KV cache: the cache's layout (include/syfi_kv.h) and its checks.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/syfi_kv.h"
#include "moe_internal.h"
#include "ptx.cuh"

namespace syfi {

constexpr int kKvPage = SYFI_KV_PAGE;

// A cache in device memory.  A block is a page's tokens of one kind (0 keys, 1 values) and head.
struct KvCache {
  uint8_t* base;
  long long page_stride;   // bytes
  int num_pages;
  int kinds;
  int heads;
};

template <int D>
__device__ __forceinline__ uint8_t* kv_block(const KvCache& c, int page, int kind, int head) {
  return c.base + page * c.page_stride + static_cast<long long>(kind * c.heads + head) * (kKvPage * (D + 4));
}

// Of the queries of one call, for every kernel that works on them.
struct KvBatch {
  const int32_t* block_table;   // [batch, max_pages]
  const int32_t* seq_lens;      // [batch]
  const int32_t* q_starts;      // [batch + 1]
  int batch, max_pages, tokens;
};

// Rows [first, first + count) of q are sequence b's new tokens, `length` its positions.  Bad tables give an empty or a shorter
// sequence, never an index outside the tensors.
struct KvSequence {
  int first, count, length;
};
__device__ __forceinline__ KvSequence kv_sequence(const KvBatch& a, int b) {
  const int lo = min(max(a.q_starts[b], 0), a.tokens), hi = min(max(a.q_starts[b + 1], lo), a.tokens);
  return {lo, hi - lo, static_cast<int>(min(static_cast<long long>(max(a.seq_lens[b], 0)), static_cast<long long>(a.max_pages) * kKvPage))};
}

// The cache's arguments as every entry point takes them; null when they are in order, else what is wrong.
inline const char* kv_cache_error(const void* base, int64_t num_pages, int64_t page_stride, int32_t kinds, int32_t heads,
                                  int32_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return "head_dim must be 64 or 128";
  if (kinds != 1 && kinds != 2) return "a cache holds keys (kinds = 1) or keys and values (kinds = 2)";
  if (heads < 1 || heads > 1024) return "kv_heads out of range";
  if (num_pages < 1 || num_pages > (1ll << 24)) return "num_pages out of range";
  if (page_stride < static_cast<int64_t>(kinds) * heads * kKvPage * (head_dim + 4) || page_stride % 16 != 0 || page_stride > (1ll << 36))
    return "page_stride is smaller than a page or no multiple of 16";
  if (!base || (reinterpret_cast<uintptr_t>(base) & 15u)) return "the cache is null or not 16-byte aligned";
  return nullptr;
}
inline bool kv_aligned(const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool kv_table_aligned(const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }   // int32, read one by one
// distance of two tokens in elements
inline bool kv_stride_ok(int64_t stride, int64_t least) { return stride >= least && stride % 8 == 0 && stride <= (1ll << 40); }

// The current device's number of SMs; 0 with the error recorded when there is none or it is no sm_100.
int kv_device_sms();

inline int kv_fail(int code, const char* msg) { return set_last_error(code, msg); }

}  // namespace syfi
