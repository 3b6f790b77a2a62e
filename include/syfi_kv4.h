/* C ABI of the paged KV cache held in 4 bits and the attention over it, in the same shared library as the MoE layer, the indexer
 * and the 8-bit cache (libsyfi_moe.so).  It is the sibling of include/syfi_kv.h with 76 instead of 132 bytes for a vector of 128:
 *
 *   bytes [num_pages, 2 (keys, values), kv_heads, 64 * (head_dim / 2 + head_dim / 16 + 4)]
 *
 * A block is 64 tokens.  It begins with head_dim / 64 planes of 64 dimensions; a plane is 64 tokens of 32 bytes, a byte the e2m1
 * codes of two neighbouring dimensions, the even one in its low half.  Then come the tokens' head_dim / 16 e4m3 group scales, one
 * for 16 dimensions, then their f32 scales.  Dimension d of token `offset` has its code in byte (d / 64) * 2048 + offset * 32 +
 * (d % 64) / 2, its group scale in byte 32 * head_dim + offset * (head_dim / 16) + d / 16, and its scale at 36 * head_dim + 4 * offset.
 * It stands for code * group scale * scale; the codes 0 .. 7 are 0, 0.5, 1, 1.5, 2, 3, 4, 6, and 8 .. 15 the same below zero.
 * `page_stride` is the distance of two pages in bytes.  A slot is page * 64 + offset.
 *
 * All pointers are DEVICE pointers, 16-byte aligned (int32 tables: 4-byte); head_dim is 64 or 128; strides of q, k, v and outputs are
 * the distance of two tokens in elements (multiples of 8), a token's heads lie side by side.  Work is enqueued on `stream` (a
 * cudaStream_t) of the CURRENT device; no call synchronises.  Every call returns SYFI_KV4_OK or an error code;
 * syfi_moe_last_error() (syfi_moe.h) has the message. */
#ifndef SYFI_KV4_H_
#define SYFI_KV4_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SYFI_KV4_OK 0
#define SYFI_KV4_ERR_INVALID 1   /* bad argument */
#define SYFI_KV4_ERR_CUDA 2      /* a CUDA call failed, no CUDA device, or not an sm_100 device */
#define SYFI_KV4_ERR_DEVICE 3    /* a kernel gave up on a bounded wait (syfi_kv4_check) */
#define SYFI_KV4_PAGE 64

/* New tokens' queries, keys and values: head norms, rotation, quantisation and the scatter into the cache in one pass.  Arguments as
 * syfi_kv_write's (syfi_kv.h), norm and rotation the same; the cache always holds keys and values.  q (with q_out) may be null with
 * q_heads = 0.  No two tokens of a call may have one slot: it may then hold some of each.
 * A head vector z (rounded to bf16 nowhere on its way) is kept as
 *   scale = max(max |z|, 1e-12) / 2688,   group scale = e4m3(max over the group of |z| / (6 scale)),
 *   code = e2m1(z / (group scale * scale)), at most 6; 0 where the group scale is 0,
 * each operation in f32, roundings to nearest, to even between two.  A vector with a NaN or an infinity is read back as NaN. */
int syfi_kv4_write(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight, const float* cos_sin,
                   const int32_t* positions, const int32_t* slots, int64_t tokens, int32_t q_heads, int32_t kv_heads,
                   int32_t head_dim, int32_t rotary_dim, int32_t interleaved, int64_t max_positions, int64_t q_stride,
                   int64_t k_stride, int64_t v_stride, int64_t q_out_stride, double eps, void* cache, int64_t num_pages,
                   int64_t page_stride, void* q_out, void* stream);

/* Rows of the cache by slot: k_out and v_out [rows, kv_heads, head_dim] (contiguous) get code * group scale * scale, rounded to bf16, or
 * in f32 where out_f32 is not 0.  A slot outside the cache (-1: not there) gives zeros.  Either output may be null. */
int syfi_kv4_read(const void* cache, int64_t num_pages, int64_t page_stride, int32_t kv_heads, int32_t head_dim,
                  const int32_t* slots, int64_t rows, int32_t out_f32, void* k_out, void* v_out, void* stream);

/* Attention of new tokens over the cache (their own keys and values included, which syfi_kv4_write has put there).  Arguments and
 * what a query sees are syfi_paged_attention's (syfi_kv.h):
 *   out = sum_j softmax_j(scale * q . key_j) * value_j;  a query that sees nothing gets zeros; rows of no sequence are left alone.
 * Positions that a query does not see do not touch its result, whatever the cache holds there.  Scales and group scales are not
 * negative.  A query, or a seen position with a scale or a key's group scale that is not finite, makes its heads' results NaN; a value's
 * group scale that is not finite those of its dimensions at least.
 * Where `scale` times a query's largest dimension, or that times a seen key's largest, is beyond f32's range, results may be NaN; where the
 * first is below 2^-110, scores are coarser than f32.
 * Sums are in f32.  A weight times its value's scale is rounded to f16 (2^-12 of it on average); one 2^-28 below the row's largest
 * may not be added, with up to 32 rows per sequence and key head on average one 2^-32 below.  Codes times group scales are exact.
 * Scratch memory by stream and by captured graph as for syfi_paged_attention, in buffers of its own. */
int syfi_kv4_attention(const void* q, int64_t q_stride, const void* cache, int64_t num_pages, int64_t page_stride,
                       const int32_t* block_table, int32_t max_pages, const int32_t* seq_lens, const int32_t* q_starts,
                       int32_t batch, int64_t tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim, double scale,
                       int32_t window, void* out, int64_t out_stride, void* stream);

/* The three calls above with their arguments, in their order, in one block of 8-byte words: pointers and integers as int64, doubles as
 * their bits. */
int syfi_kv4_write_block(const int64_t* args);
int syfi_kv4_read_block(const int64_t* args);
int syfi_kv4_attention_block(const int64_t* args);

/* Synchronises `stream` and reports whether an attention kernel gave up on a bounded wait on the current device since the last
 * check (status 401; the rows that it had not finished are NaN). */
int syfi_kv4_check(void* stream);

#ifdef __cplusplus
}
#endif

#endif  /* SYFI_KV4_H_ */
