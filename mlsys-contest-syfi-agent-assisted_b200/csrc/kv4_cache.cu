// Writing the paged KV cache in 4 bits and reading rows of it back (include/syfi_kv4.h).  Both move bytes: what they read and write once
// is their floor, so each is one pass with everything in between in registers.
#include <type_traits>

#include "kv4_internal.h"

namespace syfi {

namespace {

constexpr int kThreads = 256;
// Vectors that a group of lanes has under way.  Two instead of four: writing 8192 tokens 98 us instead of 82, reading 40,000 rows 57 instead
// of 53; eight: 53 as well.
constexpr int kWriteHeads = 4, kReadVectors = 4;
// Groups per SM that are enough to keep it busy; where four vectors each would leave fewer, a group takes one.  One and four, us: writing 300
// tokens of 32 + 2 * 8 heads of 128 9.5 and 9.4 to 10.2, 1000 15.6 and 15.6, 2000 23.8 and 21.8, 4000 44 and 34; reading 4000 rows of 8 heads
// 14.3 and 14.3, 8000 22.5 and 20.5, 20000 43 and 33.
constexpr int kFullGroups = 64;

struct Write4Args {
  const __nv_bfloat16 *q, *k, *v, *q_weight, *k_weight;
  const float* cos_sin;
  const int32_t *positions, *slots;
  __nv_bfloat16* q_out;
  long long q_stride, k_stride, v_stride, q_out_stride, max_positions;
  KvCache cache;
  int tokens, q_heads, rotary;
  float eps;
};

__device__ __forceinline__ uint4 bf16x8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void floats8(uint4 p, float (&x)[8]) {
  const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
// x / y given RN(1 / y): the product and one step with its exact remainder (Markstein), which leaves the quotient correctly rounded, so
// that a value half way between two codes goes where the division would send it.
__device__ __forceinline__ float quotient(float x, float y, float inverse) {
  const float q = x * inverse;
  return fmaf(fmaf(-q, y, x), inverse, q);
}

// A lane's eight values of a vector at `x`: eight neighbours, or four of each half.
template <int D, int PARTS>
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* x, int lane) {
  if constexpr (PARTS == 1) return *reinterpret_cast<const uint4*>(x + lane * 8);
  const uint2 low = *reinterpret_cast<const uint2*>(x + lane * 4), high = *reinterpret_cast<const uint2*>(x + D / 2 + lane * 4);
  return make_uint4(low.x, low.y, high.x, high.y);
}
template <int D, int PARTS>
__device__ __forceinline__ void store8(__nv_bfloat16* x, int lane, uint4 p) {
  if constexpr (PARTS == 1) {
    *reinterpret_cast<uint4*>(x + lane * 8) = p;
  } else {
    *reinterpret_cast<uint2*>(x + lane * 4) = make_uint2(p.x, p.y);
    *reinterpret_cast<uint2*>(x + D / 2 + lane * 4) = make_uint2(p.z, p.w);
  }
}

// How a token's rotation pairs the dimensions: neighbours, halves of the rotated part, halves of the whole vector (or no rotation at all).
enum Turn { kNeighbours, kHalves, kWholeHalves };

// A warp takes a run of neighbouring heads of one kind (queries, keys or values) of a token, D / 8 lanes per head and HEADS heads one
// after the other, whose loads are under way together and which share the token's cosines and sines.  A lane has eight neighbouring
// dimensions: a word of codes, half a group.  Its partner's in a rotation of halves come by shuffles (rotary / 2 is a multiple of eight).
// Where the whole vector is rotated by halves, or not at all, a lane has four neighbouring dimensions of each half instead: both of a pair
// are its own, and it keeps half as many cosines and sines (8192 tokens of 64 query and 2 * 8 cache heads of 128: 82 us instead of 88).
//
// The bytes take 48 us there.  What keeps it from them is the latency of a key's or value's instructions (its quotients and conversions: 67 % of the
// issue slots) with few warps to hide it, and those registers set the occupancy of the queries' warps too; four blocks to an SM, 64 registers a
// thread: with three 92 us, with five (spills) 82.  With halves of part of the dimensions four heads spill 12 bytes.
template <int D, Turn TURN, int HEADS>
__global__ void __launch_bounds__(kThreads, HEADS > 1 ? 4 : 1) kv4_write_kernel(const __grid_constant__ Write4Args a) {
  constexpr int kLanes = D / 8, kGroups = 32 / kLanes, kRun = kGroups * HEADS;
  constexpr int kParts = TURN == kWholeHalves ? 2 : 1, kEach = 8 / kParts;        // a lane's parts and the dimensions of each
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % kLanes, group = (threadIdx.x & 31) / kLanes;
  const unsigned q_runs = (a.q_heads + kRun - 1) / kRun, kv_runs = (a.cache.heads + kRun - 1) / kRun, runs = q_runs + 2 * kv_runs;
  const unsigned id = blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
  const int t = static_cast<int>(id / runs);
  if (t >= a.tokens) return;
  unsigned run = id - t * runs;
  const int which = run < q_runs ? 0 : run < q_runs + kv_runs ? 1 : 2;      // queries, keys, values; the same for the warp
  if (which > 0) run -= q_runs + (which - 1) * kv_runs;
  const int slot = which > 0 ? a.slots[t] : 0;
  if (which > 0 && (slot < 0 || slot / kKvPage >= a.cache.num_pages)) return;
  const int heads = which == 0 ? a.q_heads : a.cache.heads, first = static_cast<int>(run) * kRun + group;
  const __nv_bfloat16* const from = which == 0 ? a.q + t * a.q_stride : which == 1 ? a.k + t * a.k_stride : a.v + t * a.v_stride;
  uint4 raw[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; ++h)
    raw[h] = first + h * kGroups < heads ? load8<D, kParts>(from + (first + h * kGroups) * D, lane) : make_uint4(0u, 0u, 0u, 0u);
  // what the heads share: weights, cosines and sines
  const __nv_bfloat16* const weight = which == 0 ? a.q_weight : which == 1 ? a.k_weight : nullptr;
  float w[8];
  if (weight) floats8(load8<D, kParts>(weight, lane), w);
  const bool rotates = which < 2 && a.rotary > 0, turned = rotates && lane < a.rotary / 8;
  const int half = a.rotary / 16;               // lanes of half of the rotated dimensions
  const int partner = (threadIdx.x & 31) + (lane < half ? half : -half);
  constexpr int kTurns = TURN == kHalves ? 8 : 4;
  float cs[kTurns], sn[kTurns];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    cs[i] = 1.0f;
    sn[i] = 0.0f;
  }
  bool known = true;
  if (rotates) {
    const int position = a.positions[t];
    known = position >= 0 && position < a.max_positions;
    if (turned) {
      const float* row = a.cos_sin + (known ? position : 0) * static_cast<long long>(a.rotary) + (TURN != kHalves ? lane * 4 : (lane < half ? lane : lane - half) * 8);
#pragma unroll
      for (int i = 0; i < kTurns; i += 4) {
        const float4 c = *reinterpret_cast<const float4*>(row + i), s = *reinterpret_cast<const float4*>(row + a.rotary / 2 + i);
        cs[i] = c.x; cs[i + 1] = c.y; cs[i + 2] = c.z; cs[i + 3] = c.w;
        sn[i] = s.x; sn[i + 1] = s.y; sn[i + 2] = s.z; sn[i + 3] = s.w;
      }
      if (TURN == kHalves && lane < half) {
#pragma unroll
        for (int i = 0; i < kTurns; ++i) sn[i] = -sn[i];
      }
    }
  }
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    const int head = first + h * kGroups;
    const bool real = head < heads;
    float x[8];
    floats8(raw[h], x);
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
    if (rotates) {
      if constexpr (TURN != kHalves) {
        if (turned) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float &u = x[TURN == kNeighbours ? 2 * i : i], &v = x[TURN == kNeighbours ? 2 * i + 1 : 4 + i];
            const float turned_u = u * cs[i] - v * sn[i];
            v = v * cs[i] + u * sn[i];
            u = turned_u;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float other = __shfl_sync(0xffffffffu, x[i], partner);
          if (turned) x[i] = x[i] * cs[i] + other * sn[i];
        }
      }
    }
    if (!known) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __int_as_float(0x7fffffff);
    }
    if (which == 0) {
      if (real) store8<D, kParts>(a.q_out + t * a.q_out_stride + head * D, lane, bf16x8(x));
      continue;
    }
    // Largest magnitudes as bits: unlike the largest float they keep a NaN.  A group is in 2 * kParts lanes.
    unsigned top = 0u, tops[kParts];
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      tops[p] = 0u;
#pragma unroll
      for (int i = 0; i < kEach; ++i) tops[p] = max(tops[p], __float_as_uint(x[p * kEach + i]) & 0x7fffffffu);
#pragma unroll
      for (int d = 1; d < 2 * kParts; d <<= 1) tops[p] = max(tops[p], __shfl_xor_sync(0xffffffffu, tops[p], d));
      top = max(top, tops[p]);
    }
#pragma unroll
    for (int d = 2 * kParts; d < kLanes; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (!real) continue;
    const float largest = __uint_as_float(top);
    float scale = quotient(largest < 1e-12f ? 1e-12f : largest, 2688.0f, 1.0f / 2688.0f);
    const float six = 6.0f * scale, over_six = 1.0f / six;
    const bool finite = top < 0x7f800000u;
    uint8_t* const block = kv4_block<D>(a.cache, slot / kKvPage, which - 1, head);
    const int at = slot % kKvPage;
    uint32_t group_bytes[kParts];
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      group_bytes[p] = finite ? cvt_e4m3x2(quotient(__uint_as_float(tops[p]), six, over_six), 0.0f) & 0x7fu : 0u;
      const float unit = e4m3x2_to_float2(static_cast<uint16_t>(group_bytes[p])).x * scale, inverse = 1.0f / unit;
#pragma unroll
      for (int i = 0; i < kEach; ++i) x[p * kEach + i] = group_bytes[p] != 0u ? quotient(x[p * kEach + i], unit, inverse) : 0.0f;
      if (lane % (2 * kParts) == 0) block[Kv4Block<D>::kGroups + at * (D / kKv4Group) + p * (D / kKv4Group / 2) + lane / (2 * kParts)] = static_cast<uint8_t>(group_bytes[p]);
    }
    const uint32_t codes = cvt_e2m1x8(x);
    if constexpr (kParts == 1) {
      *reinterpret_cast<uint32_t*>(block + lane / 8 * kKv4Plane + at * 32 + lane % 8 * 4) = codes;
    } else {
#pragma unroll
      for (int p = 0; p < 2; ++p)
        *reinterpret_cast<uint16_t*>(block + (D == 128 ? p * kKv4Plane : p * 16) + at * 32 + lane * 2) = static_cast<uint16_t>(codes >> (16 * p));
    }
    if (lane == 0) *reinterpret_cast<float*>(block + Kv4Block<D>::kScales + at * 4) = finite ? scale : __int_as_float(0x7fffffff);
  }
}

// D / 8 lanes have a vector, eight dimensions each, and EACH neighbouring ones (heads of keys, then of values) of a row at a time.
// 40,000 rows of 8 key heads of 128, in bf16: 46 to 53 us, in f32 102.  The bytes take 32; rows from all over the cache bring whole sectors of 32
// bytes for 8 of group scales and 4 of a scale, 116 MB for 49, which makes it 35.  The rest is instructions: 31 million of a warp, 65 % of the
// issue slots (a lane's address arithmetic, byte loads of group scales, a scale that every lane of a vector loads).
template <int D, typename Out, int EACH>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(KvCache c, const int32_t* __restrict__ slots, unsigned rows, int first_kind, int kinds,
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
  const int at = slot % kKvPage;
  uint32_t codes[EACH], group[EACH];
  float scale[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    codes[i] = group[i] = 0u;
    scale[i] = 0.0f;
    if (there && first + i < vectors) {
      const int kind = first + i >= c.heads;
      const uint8_t* block = kv4_block<D>(c, slot / kKvPage, first_kind + kind, first + i - kind * c.heads);
      codes[i] = *reinterpret_cast<const uint32_t*>(block + lane / 8 * kKv4Plane + at * 32 + lane % 8 * 4);
      group[i] = block[Kv4Block<D>::kGroups + at * (D / kKv4Group) + lane / 2];
      scale[i] = *reinterpret_cast<const float*>(block + Kv4Block<D>::kScales + at * 4);
    }
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (first + i >= vectors) break;
    const int kind = first + i >= c.heads;
    Out* out = (first_kind + kind == 0 ? k_out : v_out) + (static_cast<long long>(row) * c.heads + first + i - kind * c.heads) * D + lane * 8;
    const uint32_t h[4] = {e2m1x2_to_half2<0>(codes[i]), e2m1x2_to_half2<1>(codes[i]), e2m1x2_to_half2<2>(codes[i]), e2m1x2_to_half2<3>(codes[i])};
    const float g = e4m3x2_to_float2(static_cast<uint16_t>(group[i])).x;
    float x[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
      x[2 * j] = f.x * g * scale[i];          // (the first product is exact)
      x[2 * j + 1] = f.y * g * scale[i];
    }
    if constexpr (sizeof(Out) == 4) {
      reinterpret_cast<float4*>(out)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(out)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      *reinterpret_cast<uint4*>(out) = bf16x8(x);
    }
  }
}

}  // namespace

}  // namespace syfi

using namespace syfi;

extern "C" int syfi_kv4_write(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight,
                              const float* cos_sin, const int32_t* positions, const int32_t* slots, int64_t tokens,
                              int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t rotary_dim, int32_t interleaved,
                              int64_t max_positions, int64_t q_stride, int64_t k_stride, int64_t v_stride, int64_t q_out_stride,
                              double eps, void* cache, int64_t num_pages, int64_t page_stride, void* q_out, void* stream) {
  if (const char* wrong = kv4_cache_error(cache, num_pages, page_stride, kv_heads, head_dim)) return kv_fail(SYFI_KV4_ERR_INVALID, wrong);
  if (tokens < 0 || q_heads < 0 || q_heads > 4096 || tokens > 0x7fffffffll / (q_heads + 2ll * kv_heads)) return kv_fail(SYFI_KV4_ERR_INVALID, "tokens or q_heads out of range");
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16 != 0) return kv_fail(SYFI_KV4_ERR_INVALID, "rotary_dim must be a multiple of 16 up to head_dim");
  if (rotary_dim > 0 && max_positions < 1) return kv_fail(SYFI_KV4_ERR_INVALID, "cos_sin has no row");
  if (!(eps >= 0.0 && eps <= 1e30)) return kv_fail(SYFI_KV4_ERR_INVALID, "eps must not be negative");
  if (tokens == 0) return SYFI_KV4_OK;
  const int64_t kv_width = static_cast<int64_t>(kv_heads) * head_dim, q_width = static_cast<int64_t>(q_heads) * head_dim;
  if (!kv_aligned(k) || !kv_aligned(v) || !kv_table_aligned(slots) || (q_heads > 0 && (!kv_aligned(q) || !kv_aligned(q_out))) ||
      (rotary_dim > 0 && (!kv_aligned(cos_sin) || !kv_table_aligned(positions))) || (q_weight && !kv_aligned(q_weight)) || (k_weight && !kv_aligned(k_weight)))
    return kv_fail(SYFI_KV4_ERR_INVALID, "a tensor argument is null or not aligned (16 bytes, int32 tables 4)");
  if (!kv_stride_ok(k_stride, kv_width) || !kv_stride_ok(v_stride, kv_width) ||
      (q_heads > 0 && (!kv_stride_ok(q_stride, q_width) || !kv_stride_ok(q_out_stride, q_width))))
    return kv_fail(SYFI_KV4_ERR_INVALID, "a token stride is smaller than the token's heads or no multiple of 8");
  const int sms = kv_device_sms();
  if (!sms) return SYFI_KV4_ERR_CUDA;
  Write4Args a;
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
  a.cache = {static_cast<uint8_t*>(cache), page_stride, static_cast<int>(num_pages), 2, kv_heads};
  a.tokens = static_cast<int>(tokens);
  a.q_heads = q_heads;
  a.rotary = rotary_dim;
  a.eps = static_cast<float>(eps);
  // One head per group of lanes while that leaves SMs idle, else a run of them.
  const int heads = q_heads + 2 * kv_heads;
  const int each = tokens * heads >= static_cast<int64_t>(sms) * kFullGroups * kWriteHeads ? kWriteHeads : 1, run_heads = 32 / (head_dim / 8) * each;
  const int64_t groups = tokens * ((q_heads + run_heads - 1) / run_heads + 2ll * ((kv_heads + run_heads - 1) / run_heads));
  const int per_block = kThreads / 32;
  const dim3 grid(static_cast<unsigned>((groups + per_block - 1) / per_block));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&](auto* kernel) { return launch_dependent(kernel, grid, dim3(kThreads), 0, st, a) == cudaSuccess; };
  const Turn turn = rotary_dim == 0 || (!interleaved && rotary_dim == head_dim) ? kWholeHalves : interleaved ? kNeighbours : kHalves;
  auto pick = [&](auto dim, auto heads_each) {
    constexpr int D = decltype(dim)::value, HEADS = decltype(heads_each)::value;
    return turn == kWholeHalves ? run(kv4_write_kernel<D, kWholeHalves, HEADS>) : turn == kNeighbours ? run(kv4_write_kernel<D, kNeighbours, HEADS>) : run(kv4_write_kernel<D, kHalves, HEADS>);
  };
  using std::integral_constant;
  const bool ok = head_dim == 128 ? (each > 1 ? pick(integral_constant<int, 128>(), integral_constant<int, kWriteHeads>()) : pick(integral_constant<int, 128>(), integral_constant<int, 1>()))
                                  : (each > 1 ? pick(integral_constant<int, 64>(), integral_constant<int, kWriteHeads>()) : pick(integral_constant<int, 64>(), integral_constant<int, 1>()));
  return ok ? SYFI_KV4_OK : kv_fail(SYFI_KV4_ERR_CUDA, "write kernel launch failed");
}

extern "C" int syfi_kv4_read(const void* cache, int64_t num_pages, int64_t page_stride, int32_t kv_heads, int32_t head_dim,
                             const int32_t* slots, int64_t rows, int32_t out_f32, void* k_out, void* v_out, void* stream) {
  if (const char* wrong = kv4_cache_error(cache, num_pages, page_stride, kv_heads, head_dim)) return kv_fail(SYFI_KV4_ERR_INVALID, wrong);
  if (rows < 0 || rows > 0x7fffffffll / 16) return kv_fail(SYFI_KV4_ERR_INVALID, "rows out of range");
  if (rows == 0 || (!k_out && !v_out)) return SYFI_KV4_OK;
  if (!kv_table_aligned(slots) || (k_out && !kv_aligned(k_out)) || (v_out && !kv_aligned(v_out))) return kv_fail(SYFI_KV4_ERR_INVALID, "a tensor argument is null or not aligned (16 bytes, int32 tables 4)");
  const int sms = kv_device_sms();
  if (!sms) return SYFI_KV4_ERR_CUDA;
  const KvCache c = {static_cast<uint8_t*>(const_cast<void*>(cache)), page_stride, static_cast<int>(num_pages), 2, kv_heads};
  const int first_kind = k_out ? 0 : 1, wanted = (k_out ? 1 : 0) + (v_out ? 1 : 0), per_block = kThreads / (head_dim / 8);
  const int each = rows * wanted * kv_heads >= static_cast<int64_t>(sms) * kFullGroups * kReadVectors ? kReadVectors : 1;
  const int64_t groups = rows * ((wanted * kv_heads + each - 1) / each);
  if (groups > 0x7fffffffll) return kv_fail(SYFI_KV4_ERR_INVALID, "rows out of range");
  const dim3 grid(static_cast<unsigned>((groups + per_block - 1) / per_block));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&](auto* kernel, auto* typed) {
    return launch_dependent(kernel, grid, dim3(kThreads), 0, st, c, slots, static_cast<unsigned>(rows), first_kind, wanted, static_cast<decltype(typed)>(k_out),
                            static_cast<decltype(typed)>(v_out)) == cudaSuccess;
  };
  float* const f32 = nullptr;
  __nv_bfloat16* const bf16 = nullptr;
  const bool ok = out_f32 ? (head_dim == 128 ? (each > 1 ? run(kv4_read_kernel<128, float, kReadVectors>, f32) : run(kv4_read_kernel<128, float, 1>, f32))
                                             : (each > 1 ? run(kv4_read_kernel<64, float, kReadVectors>, f32) : run(kv4_read_kernel<64, float, 1>, f32)))
                          : (head_dim == 128 ? (each > 1 ? run(kv4_read_kernel<128, __nv_bfloat16, kReadVectors>, bf16) : run(kv4_read_kernel<128, __nv_bfloat16, 1>, bf16))
                                             : (each > 1 ? run(kv4_read_kernel<64, __nv_bfloat16, kReadVectors>, bf16) : run(kv4_read_kernel<64, __nv_bfloat16, 1>, bf16)));
  return ok ? SYFI_KV4_OK : kv_fail(SYFI_KV4_ERR_CUDA, "read kernel launch failed");
}

extern "C" int syfi_kv4_write_block(const int64_t* args) { return kv_spread(syfi_kv4_write, args); }
extern "C" int syfi_kv4_read_block(const int64_t* args) { return kv_spread(syfi_kv4_read, args); }
extern "C" int syfi_kv4_attention_block(const int64_t* args) { return kv_spread(syfi_kv4_attention, args); }
