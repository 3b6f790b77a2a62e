// Writing the quantised paged KV cache and reading rows of it back (include/syfi_kv.h).  Both move bytes: what they read and
// write once is their floor, so each is one pass with everything in between in registers.  A lane of the write loads 8 bytes at a time and
// stores 8 or 4 (both dimensions of a rotated pair are one lane's), one of the read loads 8 and stores 16.
#include <string.h>

#include <atomic>
#include <type_traits>
#include <utility>

#include "kv_internal.h"

namespace syfi {

namespace {

constexpr int kThreads = 256;
constexpr int kWriteHeads = 4, kReadVectors = 4;   // vectors that a group of lanes has under way
// Groups per SM that are enough to keep it busy: with 16, 64, 256 a write of 600 tokens of 32 + 2 x 8 heads 11.3, 12.4, 12.5 us, of 3000 26.7,
// 26.6, 33.8; a read of 2048 rows of 2 x 8 heads 9.1, 10.2, 9.2, of 9000 15.4, 15.4, 21.4 (other memory touched in between).
constexpr int kFullGroups = 64;

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

__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A warp takes a run of neighbouring heads of one kind (queries, keys or values) of a token, D / 8 lanes per head and HEADS heads one
// after the other, whose loads are under way together and which share the token's cosines and sines.  A lane has two times four
// dimensions, chosen so that it holds both of a rotated pair: lanes below rotary / 8 have chunk l and chunk l + rotary / 8, the others two
// neighbouring chunks of what is not rotated.  Sum of squares and maximum are shuffles inside the head's lanes.
// What bounds it at many tokens is the instructions of norm, rotation and rounding beside the bytes: 8192 tokens of 64 + 2 x 8 heads of 128,
// 74 us, 4.4 TB/s.  One division per head: the eight quotients take its reciprocal and one residual each, correctly rounded as a
// division's.  Few tokens: the call itself.  Five CTAs an SM (48 registers, 36 bytes of them spilled) 79.0 us, four (63, none) 81.9, six (40, 64
// bytes) 84.0, with a flushed L2.
template <int D, bool INTERLEAVED, int HEADS>
__global__ void __launch_bounds__(kThreads, HEADS > 1 ? 5 : 1) kv_write_kernel(const __grid_constant__ WriteArgs a) {
  constexpr int kLanes = D / 8, kGroups = 32 / kLanes, kRun = kGroups * HEADS;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % kLanes, group = (threadIdx.x & 31) / kLanes;
  const unsigned q_runs = (a.q_heads + kRun - 1) / kRun, kv_runs = (a.cache.heads + kRun - 1) / kRun, runs = q_runs + a.cache.kinds * kv_runs;
  const unsigned id = blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
  const int t = static_cast<int>(id / runs);
  if (t >= a.tokens) return;
  unsigned run = id - t * runs;
  const int which = run < q_runs ? 0 : run < q_runs + kv_runs ? 1 : 2;      // queries, keys, values; the same for the warp
  if (which > 0) run -= q_runs + (which - 1) * kv_runs;
  const int slot = which > 0 ? a.slots[t] : 0;
  if (which > 0 && (slot < 0 || slot / kKvPage >= a.cache.num_pages)) return;
  const int heads = which == 0 ? a.q_heads : a.cache.heads, first = static_cast<int>(run) * kRun + group;
  const int turning = a.rotary / 8;                                         // lanes that hold rotated pairs
  const bool turned = lane < turning && which < 2;
  const bool apart = !INTERLEAVED && lane < turning;
  const int dims[2] = {apart ? 4 * lane : 8 * lane, apart ? 4 * lane + a.rotary / 2 : 8 * lane + 4};   // (8 lanes' worth of rotary lie in front of the rest)
  const __nv_bfloat16* const from = which == 0 ? a.q + t * a.q_stride : which == 1 ? a.k + t * a.k_stride : a.v + t * a.v_stride;
  uint2 raw[HEADS][2];
#pragma unroll
  for (int h = 0; h < HEADS; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      raw[h][e] = first + h * kGroups < heads ? *reinterpret_cast<const uint2*>(from + (first + h * kGroups) * D + dims[e]) : make_uint2(0u, 0u);
  // what the heads share: weights, cosines and sines (of pair i: dimensions i of both chunks, or 2 i and 2 i + 1 of both in a row)
  const __nv_bfloat16* const weight = which == 0 ? a.q_weight : which == 1 ? a.k_weight : nullptr;
  float w[8], cs[4], sn[4];
  if (weight) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint2 p = *reinterpret_cast<const uint2*>(weight + dims[e]);
      w[4 * e] = __uint_as_float(p.x << 16);
      w[4 * e + 1] = __uint_as_float(p.x & 0xffff0000u);
      w[4 * e + 2] = __uint_as_float(p.y << 16);
      w[4 * e + 3] = __uint_as_float(p.y & 0xffff0000u);
    }
  }
  bool known = true;
  if (which < 2 && a.rotary > 0) {
    const int position = a.positions[t];
    known = position >= 0 && position < a.max_positions;
    if (turned) {
      const float* row = a.cos_sin + (known ? position : 0) * static_cast<long long>(a.rotary) + lane * 4;
      const float4 c = *reinterpret_cast<const float4*>(row), s = *reinterpret_cast<const float4*>(row + a.rotary / 2);
      cs[0] = c.x; cs[1] = c.y; cs[2] = c.z; cs[3] = c.w;
      sn[0] = s.x; sn[1] = s.y; sn[2] = s.z; sn[3] = s.w;
    }
  }
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    const int head = first + h * kGroups;
    const bool real = head < heads;
    float x[8];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      x[4 * e] = __uint_as_float(raw[h][e].x << 16);
      x[4 * e + 1] = __uint_as_float(raw[h][e].x & 0xffff0000u);
      x[4 * e + 2] = __uint_as_float(raw[h][e].y << 16);
      x[4 * e + 3] = __uint_as_float(raw[h][e].y & 0xffff0000u);
    }
    if (weight) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
      for (int d = kLanes / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const float factor = rsqrtf(sum * (1.0f / D) + a.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= factor * w[i];
    }
    if (turned) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int u = INTERLEAVED ? 2 * i : i, v = INTERLEAVED ? 2 * i + 1 : i + 4;
        const float xu = x[u], xv = x[v];
        x[u] = xu * cs[i] - xv * sn[i];
        x[v] = xv * cs[i] + xu * sn[i];
      }
    }
    if (!known) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __int_as_float(0x7fffffff);
    }
    if (which == 0) {
      if (real) {
        __nv_bfloat16* const to = a.q_out + t * a.q_out_stride + head * D;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const __nv_bfloat162 lo = __floats2bfloat162_rn(x[4 * e], x[4 * e + 1]), hi = __floats2bfloat162_rn(x[4 * e + 2], x[4 * e + 3]);
          *reinterpret_cast<uint2*>(to + dims[e]) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        }
      }
      continue;
    }
    // Largest magnitude as bits: unlike the largest float it keeps a NaN.
    unsigned top = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int d = kLanes / 2; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float largest = __uint_as_float(top);
    const float scale = (largest < 1e-12f ? 1e-12f : largest) / 448.0f;
    if (!real) continue;
    // x / scale for eight x: the product with the reciprocal and one step with its exact remainder (Markstein), which leaves the quotient
    // correctly rounded, so that a value half way between two e4m3 neighbours goes where the division would send it
    const float inverse = 1.0f / scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float quotient = x[i] * inverse;
      x[i] = fmaf(fmaf(-quotient, scale, x[i]), inverse, quotient);
    }
    uint8_t* const block = kv_block<D>(a.cache, slot / kKvPage, which - 1, head);
    const int at = slot % kKvPage;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<uint32_t*>(block + at * D + dims[e]) =
          cvt_e4m3x2(x[4 * e], x[4 * e + 1]) | static_cast<uint32_t>(cvt_e4m3x2(x[4 * e + 2], x[4 * e + 3])) << 16;
    if (lane == 0) *reinterpret_cast<float*>(block + kKvPage * D + at * 4) = scale;
  }
}

// D / 8 lanes have a vector, eight dimensions each, and EACH neighbouring ones (heads of keys, then of values) of a row at a time.
// What bounds it is the bytes: 40000 rows of 2 x 8 heads of 128, 43 us, 5.8 TB/s to bf16 (91 us, 4.5 TB/s to f32).
template <int D, typename Out, int EACH>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(KvCache c, const int32_t* __restrict__ slots, unsigned rows, int first_kind, int kinds,
                                                           Out* __restrict__ k_out, Out* __restrict__ v_out) {
  constexpr int kLanes = D / 8;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % kLanes, vectors = kinds * c.heads, runs = (vectors + EACH - 1) / EACH;
  const unsigned id = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  const unsigned row = id / static_cast<unsigned>(runs);
  const int first = static_cast<int>(id - row * static_cast<unsigned>(runs)) * EACH;
  if (row >= rows) return;
  const int slot = slots[row];
  const bool there = slot >= 0 && slot / kKvPage < c.num_pages;
  uint2 bytes[EACH];
  float scale[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    bytes[i] = make_uint2(0u, 0u);
    scale[i] = 0.0f;
    if (there && first + i < vectors) {
      const int kind = first + i >= c.heads;
      const uint8_t* block = kv_block<D>(c, slot / kKvPage, first_kind + kind, first + i - kind * c.heads);
      bytes[i] = *reinterpret_cast<const uint2*>(block + slot % kKvPage * D + lane * 8);
      scale[i] = *reinterpret_cast<const float*>(block + kKvPage * D + slot % kKvPage * 4);
    }
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (first + i >= vectors) break;
    const int kind = first + i >= c.heads;
    Out* out = (first_kind + kind == 0 ? k_out : v_out) + (static_cast<long long>(row) * c.heads + first + i - kind * c.heads) * D + lane * 8;
    float x[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = e4m3x2_to_float2(static_cast<uint16_t>((j < 2 ? bytes[i].x : bytes[i].y) >> (16 * (j % 2))));
      x[2 * j] = f.x * scale[i];
      x[2 * j + 1] = f.y * scale[i];
    }
    if constexpr (sizeof(Out) == 4) {
      reinterpret_cast<float4*>(out)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(out)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      *reinterpret_cast<uint4*>(out) = pack8(x);
    }
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
  if (tokens < 0 || q_heads < 0 || q_heads > 4096 || tokens > 0x7fffffffll / (q_heads + 2ll * kv_heads)) return kv_fail(SYFI_KV_ERR_INVALID, "tokens or q_heads out of range");
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
  const int sms = kv_device_sms();
  if (!sms) return SYFI_KV_ERR_CUDA;
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
  // One head per group of lanes while that leaves SMs idle, else a run of them.
  const int heads = q_heads + kinds * kv_heads;
  const int each = tokens * heads >= static_cast<int64_t>(sms) * kFullGroups * kWriteHeads ? kWriteHeads : 1, run_heads = 32 / (head_dim / 8) * each;
  const int64_t groups = tokens * ((q_heads + run_heads - 1) / run_heads + static_cast<int64_t>(kinds) * ((kv_heads + run_heads - 1) / run_heads));
  const int per_block = kThreads / 32;
  const dim3 grid(static_cast<unsigned>((groups + per_block - 1) / per_block));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&](auto* kernel) { return launch_dependent(kernel, grid, dim3(kThreads), 0, st, a) == cudaSuccess; };
  const bool ok = head_dim == 128 ? (interleaved ? (each > 1 ? run(kv_write_kernel<128, true, kWriteHeads>) : run(kv_write_kernel<128, true, 1>))
                                                 : (each > 1 ? run(kv_write_kernel<128, false, kWriteHeads>) : run(kv_write_kernel<128, false, 1>)))
                                  : (interleaved ? (each > 1 ? run(kv_write_kernel<64, true, kWriteHeads>) : run(kv_write_kernel<64, true, 1>))
                                                 : (each > 1 ? run(kv_write_kernel<64, false, kWriteHeads>) : run(kv_write_kernel<64, false, 1>)));
  return ok ? SYFI_KV_OK : kv_fail(SYFI_KV_ERR_CUDA, "write kernel launch failed");
}

extern "C" int syfi_kv_read(const void* cache, int64_t num_pages, int64_t page_stride, int32_t kinds, int32_t kv_heads,
                            int32_t head_dim, const int32_t* slots, int64_t rows, int32_t out_f32, void* k_out, void* v_out,
                            void* stream) {
  if (const char* wrong = kv_cache_error(cache, num_pages, page_stride, kinds, kv_heads, head_dim)) return kv_fail(SYFI_KV_ERR_INVALID, wrong);
  if (rows < 0 || rows > 0x7fffffffll / 16) return kv_fail(SYFI_KV_ERR_INVALID, "rows out of range");
  if (kinds == 1 && v_out) return kv_fail(SYFI_KV_ERR_INVALID, "this cache holds no values");
  if (rows == 0 || (!k_out && !v_out)) return SYFI_KV_OK;
  if (!kv_table_aligned(slots) || (k_out && !kv_aligned(k_out)) || (v_out && !kv_aligned(v_out))) return kv_fail(SYFI_KV_ERR_INVALID, "a tensor argument is null or not aligned (16 bytes, int32 tables 4)");
  const int sms = kv_device_sms();
  if (!sms) return SYFI_KV_ERR_CUDA;
  const KvCache c = {static_cast<uint8_t*>(const_cast<void*>(cache)), page_stride, static_cast<int>(num_pages), kinds, kv_heads};
  const int first_kind = k_out ? 0 : 1, wanted = (k_out ? 1 : 0) + (v_out ? 1 : 0), per_block = kThreads / (head_dim / 8);
  const int each = rows * wanted * kv_heads >= static_cast<int64_t>(sms) * kFullGroups * kReadVectors ? kReadVectors : 1;
  const int64_t groups = rows * ((wanted * kv_heads + each - 1) / each);
  if (groups > 0x7fffffffll) return kv_fail(SYFI_KV_ERR_INVALID, "rows out of range");
  const dim3 grid(static_cast<unsigned>((groups + per_block - 1) / per_block));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&](auto* kernel, auto* typed) {
    return launch_dependent(kernel, grid, dim3(kThreads), 0, st, c, slots, static_cast<unsigned>(rows), first_kind, wanted, static_cast<decltype(typed)>(k_out),
                            static_cast<decltype(typed)>(v_out)) == cudaSuccess;
  };
  float* const f32 = nullptr;
  __nv_bfloat16* const bf16 = nullptr;
  const bool ok = out_f32 ? (head_dim == 128 ? (each > 1 ? run(kv_read_kernel<128, float, kReadVectors>, f32) : run(kv_read_kernel<128, float, 1>, f32))
                                             : (each > 1 ? run(kv_read_kernel<64, float, kReadVectors>, f32) : run(kv_read_kernel<64, float, 1>, f32)))
                          : (head_dim == 128 ? (each > 1 ? run(kv_read_kernel<128, __nv_bfloat16, kReadVectors>, bf16) : run(kv_read_kernel<128, __nv_bfloat16, 1>, bf16))
                                             : (each > 1 ? run(kv_read_kernel<64, __nv_bfloat16, kReadVectors>, bf16) : run(kv_read_kernel<64, __nv_bfloat16, 1>, bf16)));
  return ok ? SYFI_KV_OK : kv_fail(SYFI_KV_ERR_CUDA, "read kernel launch failed");
}

// ---------------------------------------------------------------- the entry points with their arguments in one block
namespace {
template <typename T>
T at(const int64_t* args, int i) {
  if constexpr (std::is_pointer_v<T>) return reinterpret_cast<T>(args[i]);
  else if constexpr (std::is_same_v<T, double>) {
    double v;
    memcpy(&v, args + i, sizeof(v));
    return v;
  } else return static_cast<T>(args[i]);
}
template <typename T>
bool fits(int64_t word) { return !std::is_same_v<T, int32_t> || word == static_cast<int32_t>(word); }
template <typename... Args, size_t... I>
int spread(int (*fn)(Args...), const int64_t* args, std::index_sequence<I...>) {
  if (!(fits<Args>(args[I]) && ...)) return kv_fail(SYFI_KV_ERR_INVALID, "an argument does not fit in 32 bits");
  return fn(at<Args>(args, static_cast<int>(I))...);
}
template <typename... Args>
int spread(int (*fn)(Args...), const int64_t* args) {
  return args ? spread(fn, args, std::index_sequence_for<Args...>()) : kv_fail(SYFI_KV_ERR_INVALID, "no arguments");
}
}  // namespace

extern "C" int syfi_kv_write_block(const int64_t* args) { return spread(syfi_kv_write, args); }
extern "C" int syfi_kv_read_block(const int64_t* args) { return spread(syfi_kv_read, args); }
extern "C" int syfi_paged_attention_block(const int64_t* args) { return spread(syfi_paged_attention, args); }
