// Attention of new tokens over the quantised paged KV cache (include/syfi_kv.h).
//
//   x_j = scale * kscale_j * sum_d q_d k_jd,   m = max x_j,   l = sum exp(x_j - m),   out_d = sum exp(x_j - m) vscale_j v_jd / l
// over the visible positions j, in one pass over the cache: m, l and the sum are corrected by exp(m_old - m_new) when m grows.
#include "kv_internal.h"

namespace syfi {

namespace {

constexpr int kWarps = 4;

// One warp per query and head.  A lane has two of a page's 64 tokens while the scores are made and D / 32 dimensions while the
// values are added up.
template <int D>
__global__ void __launch_bounds__(kWarps * 32)
attention_rows_kernel(const __nv_bfloat16* __restrict__ q, long long q_stride, KvCache cache, KvBatch batch, int q_heads,
                      float scale_log2, int window, __nv_bfloat16* __restrict__ out, long long out_stride) {
  __shared__ float s_q[kWarps][D], s_p[kWarps][kKvPage];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long id = static_cast<long long>(blockIdx.x) * kWarps + warp;
  if (id >= static_cast<long long>(batch.tokens) * q_heads) return;
  const int t = static_cast<int>(id / q_heads), head = static_cast<int>(id - static_cast<long long>(t) * q_heads);
  int b = -1;
  KvSequence s = {};
  for (int at = 0; at < batch.batch && b < 0; at += 32) {
    KvSequence mine = {};
    if (at + lane < batch.batch) mine = kv_sequence(batch, at + lane);
    const unsigned holds = __ballot_sync(0xffffffffu, t >= mine.first && t < mine.first + mine.count);
    if (holds != 0u) b = at + __ffs(holds) - 1;
  }
  if (b < 0) return;
  s = kv_sequence(batch, b);
  const int position = s.length - s.count + (t - s.first);
  const int low = window > 0 ? max(position - window + 1, 0) : 0;
  const int kv_head = head / (q_heads / cache.heads);
  for (int d = lane; d < D; d += 32) s_q[warp][d] = __bfloat162float(q[t * q_stride + head * D + d]);
  __syncwarp();
  float m = -INFINITY, l = 0.0f, acc[D / 32] = {};
  for (int page = low / kKvPage; page * kKvPage <= position; ++page) {
    const int at = batch.block_table[static_cast<long long>(b) * batch.max_pages + page];
    if (at < 0 || at >= cache.num_pages) continue;
    const uint8_t* keys = kv_block<D>(cache, at, 0, kv_head);
    const uint8_t* values = kv_block<D>(cache, at, 1, kv_head);
    float x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int token = lane + 32 * i, j = page * kKvPage + token;
      x[i] = -INFINITY;
      if (j >= low && j <= position) {
        float sum = 0.0f;
        for (int d = 0; d < D; d += 16) {
          const uint4 p = *reinterpret_cast<const uint4*>(keys + token * D + d);
          const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 f = e4m3x2_to_float2(static_cast<uint16_t>(w[e / 2] >> (16 * (e % 2))));
            sum = fmaf(s_q[warp][d + 2 * e], f.x, fmaf(s_q[warp][d + 2 * e + 1], f.y, sum));
          }
        }
        x[i] = sum * *reinterpret_cast<const float*>(keys + kKvPage * D + token * 4) * scale_log2;
      }
    }
    float top = fmaxf(x[0], x[1]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float m_new = fmaxf(m, top), reference = m_new == -INFINITY ? 0.0f : m_new;
    const float fade = exp2f(m - reference);
    l *= fade;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] *= fade;
    m = m_new;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float p = exp2f(x[i] - reference);
      l += p;
      s_p[warp][lane + 32 * i] = p;
    }
    __syncwarp();
    const int first = max(low - page * kKvPage, 0), last = min(position - page * kKvPage, kKvPage - 1);
    for (int token = first; token <= last; ++token) {
      const float p = s_p[warp][token] * *reinterpret_cast<const float*>(values + kKvPage * D + token * 4);
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const float2 f = e4m3x2_to_float2(*reinterpret_cast<const uint16_t*>(values + token * D + i * 64 + lane * 2));
        acc[2 * i] = fmaf(p, f.x, acc[2 * i]);
        acc[2 * i + 1] = fmaf(p, f.y, acc[2 * i + 1]);
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
    *reinterpret_cast<__nv_bfloat162*>(out + t * out_stride + head * D + i * 64 + lane * 2) =
        __floats2bfloat162_rn(acc[2 * i] * inv, acc[2 * i + 1] * inv);
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
  if (tokens < 0 || tokens * q_heads > 0x3fffffffll) return kv_fail(SYFI_KV_ERR_INVALID, "tokens out of range");
  if (max_pages < 1 || max_pages > (1 << 20)) return kv_fail(SYFI_KV_ERR_INVALID, "max_pages (block table width) out of range");
  if (window < 0) return kv_fail(SYFI_KV_ERR_INVALID, "window must not be negative");
  if (!(scale > -1e30 && scale < 1e30)) return kv_fail(SYFI_KV_ERR_INVALID, "scale is not a finite float");
  if (batch == 0 || tokens == 0) return SYFI_KV_OK;
  if (!kv_aligned(q) || !kv_aligned(out) || !kv_table_aligned(block_table) || !kv_table_aligned(seq_lens) || !kv_table_aligned(q_starts))
    return kv_fail(SYFI_KV_ERR_INVALID, "a tensor argument is null or not aligned (16 bytes, int32 tables 4)");
  const int64_t width = static_cast<int64_t>(q_heads) * head_dim;
  if (!kv_stride_ok(q_stride, width) || !kv_stride_ok(out_stride, width))
    return kv_fail(SYFI_KV_ERR_INVALID, "a token stride is smaller than the token's heads or no multiple of 8");
  if (!kv_device_sms()) return SYFI_KV_ERR_CUDA;
  const KvCache c = {static_cast<uint8_t*>(const_cast<void*>(cache)), page_stride, static_cast<int>(num_pages), 2, kv_heads};
  const KvBatch batch_args = {block_table, seq_lens, q_starts, batch, max_pages, static_cast<int>(tokens)};
  const float scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  const unsigned grid = static_cast<unsigned>((tokens * q_heads + kWarps - 1) / kWarps);
  auto* kernel = head_dim == 128 ? attention_rows_kernel<128> : attention_rows_kernel<64>;
  kernel<<<grid, kWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const __nv_bfloat16*>(q), q_stride, c, batch_args, q_heads,
                                                                      scale_log2, window, static_cast<__nv_bfloat16*>(out), out_stride);
  return cudaGetLastError() == cudaSuccess ? SYFI_KV_OK : kv_fail(SYFI_KV_ERR_CUDA, "attention kernel launch failed");
}
