// Writing the quantised paged KV cache and reading rows of it back (include/syfi_kv.h).  Both move bytes: what they read and
// write once is their floor, so each is one pass with 16-byte accesses and everything in between in registers.
#include <atomic>

#include "kv_internal.h"

namespace syfi {

namespace {

constexpr int kThreads = 256;

struct WriteArgs {
  const __nv_bfloat16 *q, *k, *v, *q_weight, *k_weight;
  const float* cos_sin;
  const int32_t *positions, *slots;
  __nv_bfloat16* q_out;
  long long q_stride, k_stride, v_stride, q_out_stride, max_positions;
  KvCache cache;
  int tokens, q_heads, rotary;
  float eps;
};

__device__ __forceinline__ void unpack8(const uint4& p, float (&x)[8]) {
  const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// D / 8 lanes have a head vector, eight dimensions each: sum of squares and maximum are shuffles inside the group, the other
// half of a rotated pair comes from the lane rotary / 16 away.
template <int D, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(WriteArgs a) {
  constexpr int kLanes = D / 8;
  const int lane = threadIdx.x % kLanes;
  const int heads = a.q_heads + a.cache.kinds * a.cache.heads;
  const long long id = static_cast<long long>(blockIdx.x) * (kThreads / kLanes) + threadIdx.x / kLanes;
  const bool inside = id < static_cast<long long>(a.tokens) * heads;
  const int t = inside ? static_cast<int>(id / heads) : 0, head = inside ? static_cast<int>(id - static_cast<long long>(t) * heads) : 0;
  const bool is_q = head < a.q_heads;
  const int kv = head - a.q_heads, kind = is_q ? 0 : kv / a.cache.heads, kv_head = kv - kind * a.cache.heads;
  const int slot = is_q ? 0 : a.slots[t];
  const bool active = inside && (is_q || (slot >= 0 && slot / kKvPage < a.cache.num_pages));
  float x[8] = {};
  if (active) {
    const __nv_bfloat16* from = is_q ? a.q + t * a.q_stride + head * D
                                     : (kind == 0 ? a.k + t * a.k_stride : a.v + t * a.v_stride) + kv_head * D;
    unpack8(*reinterpret_cast<const uint4*>(from + lane * 8), x);
  }
  if (kind == 0) {       // (the same for all lanes of a group; groups of one warp may differ, so the shuffles name the group)
    const unsigned mask = (kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1u)) << ((threadIdx.x & 31) / kLanes * kLanes);
    const __nv_bfloat16* weight = is_q ? a.q_weight : a.k_weight;
    if (weight) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
      for (int d = kLanes / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(mask, sum, d);
      const float factor = rsqrtf(sum / D + a.eps);
      float w[8];
      unpack8(*reinterpret_cast<const uint4*>(weight + lane * 8), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= factor * w[i];
    }
    if (a.rotary > 0) {
      const int position = a.positions[t];
      const bool known = position >= 0 && position < a.max_positions;
      const float* row = a.cos_sin + (known ? position : 0) * static_cast<long long>(a.rotary);
      const int half = a.rotary / 16;                    // lanes that hold the first halves of the pairs
      const bool turned = lane < 2 * half;
      if constexpr (INTERLEAVED) {
        if (turned) {
          const float4 c = *reinterpret_cast<const float4*>(row + lane * 4), s = *reinterpret_cast<const float4*>(row + a.rotary / 2 + lane * 4);
          const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float u = x[2 * i], v = x[2 * i + 1];
            x[2 * i] = u * cs[i] - v * sn[i];
            x[2 * i + 1] = v * cs[i] + u * sn[i];
          }
        }
      } else {
        const bool second = lane >= half;
        const int partner = (threadIdx.x & 31) / kLanes * kLanes + (!turned ? lane : second ? lane - half : lane + half);
        float other[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(mask, x[i], partner);
        if (turned) {
          const int at = (second ? lane - half : lane) * 8;
#pragma unroll
          for (int j = 0; j < 8; j += 4) {
            const float4 c = *reinterpret_cast<const float4*>(row + at + j), s = *reinterpret_cast<const float4*>(row + a.rotary / 2 + at + j);
            const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j + i] = x[j + i] * cs[i] + (second ? other[j + i] : -other[j + i]) * sn[i];
          }
        }
      }
      if (!known) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __int_as_float(0x7fffffff);
      }
    }
  }
  if (is_q) {
    if (active) *reinterpret_cast<uint4*>(a.q_out + t * a.q_out_stride + head * D + lane * 8) = pack8(x);
    return;
  }
  // Largest magnitude as bits: unlike the largest float it keeps a NaN.
  unsigned top = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  const unsigned mask = (kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1u)) << ((threadIdx.x & 31) / kLanes * kLanes);
#pragma unroll
  for (int d = kLanes / 2; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(mask, top, d));
  const float largest = __uint_as_float(top);
  const float scale = (largest < 1e-12f ? 1e-12f : largest) / 448.0f;
  if (!active) return;
  uint32_t bytes[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    bytes[i] = cvt_e4m3x2(x[4 * i] / scale, x[4 * i + 1] / scale) | static_cast<uint32_t>(cvt_e4m3x2(x[4 * i + 2] / scale, x[4 * i + 3] / scale)) << 16;
  uint8_t* block = kv_block<D>(a.cache, slot / kKvPage, kind, kv_head);
  const int at = slot % kKvPage;
  *reinterpret_cast<uint2*>(block + at * D + lane * 8) = make_uint2(bytes[0], bytes[1]);
  if (lane == 0) *reinterpret_cast<float*>(block + kKvPage * D + at * 4) = scale;
}

// Sixteen dimensions per lane.
template <int D, typename Out>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(KvCache c, const int32_t* __restrict__ slots, long long vectors,
                                                           Out* __restrict__ k_out, Out* __restrict__ v_out) {
  constexpr int kLanes = D / 16;
  const long long id = static_cast<long long>(blockIdx.x) * (kThreads / kLanes) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  if (id >= vectors) return;
  const int per_row = c.kinds * c.heads;
  const long long row = id / per_row;
  const int which = static_cast<int>(id - row * per_row), kind = which / c.heads, head = which - kind * c.heads;
  Out* out = kind == 0 ? k_out : v_out;
  if (!out) return;
  out += (row * c.heads + head) * D + lane * 16;
  const int slot = slots[row];
  float x[16] = {};
  if (slot >= 0 && slot / kKvPage < c.num_pages) {
    const uint8_t* block = kv_block<D>(c, slot / kKvPage, kind, head);
    const int at = slot % kKvPage;
    const uint4 p = *reinterpret_cast<const uint4*>(block + at * D + lane * 16);
    const float scale = *reinterpret_cast<const float*>(block + kKvPage * D + at * 4);
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = e4m3x2_to_float2(static_cast<uint16_t>(w[i / 2] >> (16 * (i % 2))));
      x[2 * i] = f.x * scale;
      x[2 * i + 1] = f.y * scale;
    }
  }
  if constexpr (sizeof(Out) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(out)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  } else {
    const float lo[8] = {x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]}, hi[8] = {x[8], x[9], x[10], x[11], x[12], x[13], x[14], x[15]};
    reinterpret_cast<uint4*>(out)[0] = pack8(lo);
    reinterpret_cast<uint4*>(out)[1] = pack8(hi);
  }
}

std::atomic<int> g_sms[64];   // 0: not asked yet

}  // namespace

int kv_device_sms() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    kv_fail(SYFI_KV_ERR_CUDA, "no current CUDA device: this library has no CPU path");
    return 0;
  }
  int sms = g_sms[dev].load(std::memory_order_relaxed);
  if (sms == 0) {
    int major = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess || major != 10 ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
      kv_fail(SYFI_KV_ERR_CUDA, "this library is built for sm_100a (B200) only");
      return 0;
    }
    g_sms[dev].store(sms, std::memory_order_relaxed);
  }
  return sms;
}

}  // namespace syfi

using namespace syfi;

extern "C" int syfi_kv_write(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight,
                             const float* cos_sin, const int32_t* positions, const int32_t* slots, int64_t tokens,
                             int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t rotary_dim, int32_t interleaved,
                             int64_t max_positions, int64_t q_stride, int64_t k_stride, int64_t v_stride, int64_t q_out_stride,
                             double eps, void* cache, int64_t num_pages, int64_t page_stride, int32_t kinds, void* q_out,
                             void* stream) {
  if (const char* wrong = kv_cache_error(cache, num_pages, page_stride, kinds, kv_heads, head_dim)) return kv_fail(SYFI_KV_ERR_INVALID, wrong);
  if (tokens < 0 || q_heads < 0 || q_heads > 4096 || tokens * (q_heads + 2ll * kv_heads) > 0x7fffffffll) return kv_fail(SYFI_KV_ERR_INVALID, "tokens or q_heads out of range");
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16 != 0) return kv_fail(SYFI_KV_ERR_INVALID, "rotary_dim must be a multiple of 16 up to head_dim");
  if (rotary_dim > 0 && max_positions < 1) return kv_fail(SYFI_KV_ERR_INVALID, "cos_sin has no row");
  if (!(eps >= 0.0 && eps <= 1e30)) return kv_fail(SYFI_KV_ERR_INVALID, "eps must not be negative");
  if (tokens == 0) return SYFI_KV_OK;
  const int64_t kv_width = static_cast<int64_t>(kv_heads) * head_dim, q_width = static_cast<int64_t>(q_heads) * head_dim;
  if (!kv_aligned(k) || !kv_table_aligned(slots) || (kinds == 2 && !kv_aligned(v)) || (q_heads > 0 && (!kv_aligned(q) || !kv_aligned(q_out))) ||
      (rotary_dim > 0 && (!kv_aligned(cos_sin) || !kv_table_aligned(positions))) || (q_weight && !kv_aligned(q_weight)) || (k_weight && !kv_aligned(k_weight)))
    return kv_fail(SYFI_KV_ERR_INVALID, "a tensor argument is null or not aligned (16 bytes, int32 tables 4)");
  if (!kv_stride_ok(k_stride, kv_width) || (kinds == 2 && !kv_stride_ok(v_stride, kv_width)) ||
      (q_heads > 0 && (!kv_stride_ok(q_stride, q_width) || !kv_stride_ok(q_out_stride, q_width))))
    return kv_fail(SYFI_KV_ERR_INVALID, "a token stride is smaller than the token's heads or no multiple of 8");
  if (!kv_device_sms()) return SYFI_KV_ERR_CUDA;
  WriteArgs a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.k = static_cast<const __nv_bfloat16*>(k);
  a.v = static_cast<const __nv_bfloat16*>(v);
  a.q_weight = static_cast<const __nv_bfloat16*>(q_weight);
  a.k_weight = static_cast<const __nv_bfloat16*>(k_weight);
  a.cos_sin = cos_sin;
  a.positions = positions;
  a.slots = slots;
  a.q_out = static_cast<__nv_bfloat16*>(q_out);
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_out_stride = q_out_stride;
  a.max_positions = max_positions;
  a.cache = {static_cast<uint8_t*>(cache), page_stride, static_cast<int>(num_pages), kinds, kv_heads};
  a.tokens = static_cast<int>(tokens);
  a.q_heads = q_heads;
  a.rotary = rotary_dim;
  a.eps = static_cast<float>(eps);
  const long long vectors = tokens * (q_heads + static_cast<long long>(kinds) * kv_heads);
  const int per_block = kThreads / (head_dim / 8);
  const unsigned grid = static_cast<unsigned>((vectors + per_block - 1) / per_block);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) {
    if (interleaved) kv_write_kernel<128, true><<<grid, kThreads, 0, st>>>(a);
    else kv_write_kernel<128, false><<<grid, kThreads, 0, st>>>(a);
  } else {
    if (interleaved) kv_write_kernel<64, true><<<grid, kThreads, 0, st>>>(a);
    else kv_write_kernel<64, false><<<grid, kThreads, 0, st>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? SYFI_KV_OK : kv_fail(SYFI_KV_ERR_CUDA, "write kernel launch failed");
}

extern "C" int syfi_kv_read(const void* cache, int64_t num_pages, int64_t page_stride, int32_t kinds, int32_t kv_heads,
                            int32_t head_dim, const int32_t* slots, int64_t rows, int32_t out_f32, void* k_out, void* v_out,
                            void* stream) {
  if (const char* wrong = kv_cache_error(cache, num_pages, page_stride, kinds, kv_heads, head_dim)) return kv_fail(SYFI_KV_ERR_INVALID, wrong);
  if (rows < 0 || rows > 0x7fffffffll / 16) return kv_fail(SYFI_KV_ERR_INVALID, "rows out of range");
  if (kinds == 1 && v_out) return kv_fail(SYFI_KV_ERR_INVALID, "this cache holds no values");
  if (rows == 0 || (!k_out && !v_out)) return SYFI_KV_OK;
  if (!kv_table_aligned(slots) || (k_out && !kv_aligned(k_out)) || (v_out && !kv_aligned(v_out))) return kv_fail(SYFI_KV_ERR_INVALID, "a tensor argument is null or not aligned (16 bytes, int32 tables 4)");
  if (!kv_device_sms()) return SYFI_KV_ERR_CUDA;
  const KvCache c = {static_cast<uint8_t*>(const_cast<void*>(cache)), page_stride, static_cast<int>(num_pages), kinds, kv_heads};
  const long long vectors = static_cast<long long>(rows) * kinds * kv_heads;
  const int per_block = kThreads / (head_dim / 16);
  const long long blocks = (vectors + per_block - 1) / per_block;
  if (blocks > 0x7fffffffll) return kv_fail(SYFI_KV_ERR_INVALID, "rows out of range");
  const unsigned grid = static_cast<unsigned>(blocks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&](auto* kernel, auto* typed) {
    kernel<<<grid, kThreads, 0, st>>>(c, slots, vectors, static_cast<decltype(typed)>(k_out), static_cast<decltype(typed)>(v_out));
  };
  if (out_f32) {
    if (head_dim == 128) run(kv_read_kernel<128, float>, static_cast<float*>(nullptr));
    else run(kv_read_kernel<64, float>, static_cast<float*>(nullptr));
  } else {
    if (head_dim == 128) run(kv_read_kernel<128, __nv_bfloat16>, static_cast<__nv_bfloat16*>(nullptr));
    else run(kv_read_kernel<64, __nv_bfloat16>, static_cast<__nv_bfloat16*>(nullptr));
  }
  return cudaGetLastError() == cudaSuccess ? SYFI_KV_OK : kv_fail(SYFI_KV_ERR_CUDA, "read kernel launch failed");
}
