/* C ABI of the quantised paged KV cache and the attention over it, in the same shared library as the MoE layer and the
 * indexer (libsyfi_moe.so).  The cache has the layout of the indexer's key cache, for keys and values of any number of
 * heads:
 *
 *   bytes [num_pages, kinds, kv_heads, 64 * (head_dim + 4)]
 *
 * kinds = 2: keys, then values; kinds = 1: keys only (with one head of 128 dimensions this is the cache that
 * syfi_dsa_topk_indexer reads).  A block is 64 tokens of head_dim e4m3 bytes each, then the tokens' 64 f32 scales: token
 * `offset` of a page has head_dim bytes at offset * head_dim and its scale at 64 * head_dim + 4 * offset; it stands for
 * byte value * scale.  `page_stride` is the distance of two pages in bytes (a page of a layer may be a slice of a page
 * of all layers).  A slot is page * 64 + offset.
 *
 * All pointers are DEVICE pointers, 16-byte aligned (int32 tables: 4-byte); head_dim is 64 or 128; strides of q, k, v and outputs are the distance
 * of two tokens in elements (multiples of 8), a token's heads lie side by side.  Work is enqueued on `stream` (a
 * cudaStream_t) of the CURRENT device; no call synchronises.  Every call returns SYFI_KV_OK or an error code;
 * syfi_moe_last_error() (syfi_moe.h) has the message. */
#ifndef SYFI_KV_H_
#define SYFI_KV_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SYFI_KV_OK 0
#define SYFI_KV_ERR_INVALID 1   /* bad argument */
#define SYFI_KV_ERR_CUDA 2      /* a CUDA call failed, no CUDA device, or not an sm_100 device */
#define SYFI_KV_ERR_DEVICE 3    /* a kernel gave up on a bounded wait (syfi_kv_check) */
#define SYFI_KV_PAGE 64

/* New tokens' queries, keys and values: head norms, rotation, quantisation and the scatter into the cache in one pass.
 *   q [tokens, q_heads, head_dim], k and v [tokens, kv_heads, head_dim]: bf16.  q (with q_out) may be null with q_heads = 0,
 *       v is null where kinds = 1.
 *   q_weight, k_weight: bf16 [head_dim] or null; y = x / sqrt(mean(x^2) + eps) * weight over the dimensions of a head, in f32
 *       (a head whose sum of squares is beyond that becomes zeros).
 *   cos_sin: f32 [max_positions, rotary_dim] (rotary_dim / 2 cosines, then as many sines) or null with rotary_dim = 0;
 *       rotary_dim is a multiple of 16 up to head_dim.  The first rotary_dim dimensions of q and k are turned by the row of
 *       the token's position: (a, b) -> (a cos - b sin, b cos + a sin), pair i being the dimensions (i, i + rotary_dim / 2),
 *       or (2 i, 2 i + 1) where `interleaved` is not 0.  A position outside the table gives NaN.
 *   positions: int32 [tokens] (may be null with rotary_dim = 0).
 *   slots: int32 [tokens]: where a token's keys and values go; a slot outside the cache (-1: padding) is not written.  No two
 *       tokens of a call may have one slot: its scale may then be one's and its bytes the other's.
 *   q_out: bf16 [tokens, q_heads, head_dim], may be q itself.
 * A written head vector z (rounded to bf16 nowhere on its way) has the scale max(max|z|, 1e-12) / 448 and the bytes
 * e4m3(z / scale), rounded to nearest; one with a NaN or an infinity is read back as NaN. */
int syfi_kv_write(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight, const float* cos_sin,
                  const int32_t* positions, const int32_t* slots, int64_t tokens, int32_t q_heads, int32_t kv_heads,
                  int32_t head_dim, int32_t rotary_dim, int32_t interleaved, int64_t max_positions, int64_t q_stride,
                  int64_t k_stride, int64_t v_stride, int64_t q_out_stride, double eps, void* cache, int64_t num_pages,
                  int64_t page_stride, int32_t kinds, void* q_out, void* stream);

/* Rows of the cache by slot: k_out and v_out [rows, kv_heads, head_dim] (contiguous) get byte value * scale, rounded to bf16, or
 * in f32 where out_f32 is not 0.  A slot outside the cache (-1: not there, as in the indexer's result) gives zeros.
 * v_out is null where kinds = 1, and either may be null when it is not wanted. */
int syfi_kv_read(const void* cache, int64_t num_pages, int64_t page_stride, int32_t kinds, int32_t kv_heads, int32_t head_dim,
                 const int32_t* slots, int64_t rows, int32_t out_f32, void* k_out, void* v_out, void* stream);

/* Attention of new tokens over the cache (their own keys and values included, which syfi_kv_write has put there).
 *   q, out: bf16 [tokens, q_heads, head_dim]; query head h uses key head h / (q_heads / kv_heads).
 *   block_table: int32 [batch, max_pages]: cache page of every 64 positions of a sequence.  Positions of an entry outside the
 *       cache (negative: evicted) are not there.
 *   seq_lens: int32 [batch]: positions of each sequence, at most 64 * max_pages of which count.
 *   q_starts: int32 [batch + 1]: sequence b's new tokens are rows q_starts[b] .. q_starts[b + 1] - 1 of q, its last positions.
 *       Rows of no sequence are left alone.
 * The query at position p sees the positions j <= p that are there, with window > 0 only those with j > p - window:
 *   out = sum_j softmax_j(scale * q . key_j) * value_j;  a query that sees nothing gets zeros.
 * Positions that a query does not see do not touch its result, whatever the cache holds there.  Scales are not negative.  A
 * query or a seen position that is not finite makes its heads' results NaN (a NaN in some dimensions of a value: those, or all).
 * Sums are in f32.  A weight is rounded to f16 (2^-12 of it on average); one 2^-32 below the row's largest may not be added, nor,
 * with few rows, one whose value is 2^-32 below the row's largest.  With more than 16 rows per sequence and key head on average
 * q is held to 2^-17 of its row's largest dimension.
 * There the product of a query and a key is formed with the query's largest dimension brought to 2^7 .. 2^8 (by 2^120 at most); where that
 * product is beyond f32's range, results may be NaN.
 * Calls on different streams may run at the same time: every stream has a scratch buffer of its own (up to 45 MB), which
 * grows on demand (that waits for the device).  Up to eight streams of a device hold one; a ninth waits for the device and takes
 * over the least recently used.  A captured graph has buffers of its own, one for each stream that was captured into it, until it is
 * destroyed: it may be replayed beside anything but itself. */
int syfi_paged_attention(const void* q, int64_t q_stride, const void* cache, int64_t num_pages, int64_t page_stride,
                         const int32_t* block_table, int32_t max_pages, const int32_t* seq_lens, const int32_t* q_starts,
                         int32_t batch, int64_t tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim, double scale,
                         int32_t window, void* out, int64_t out_stride, void* stream);

/* The three calls above with their arguments, in their order, in one block of 8-byte words: pointers and integers as int64, doubles as
 * their bits.  For hosts whose foreign function interface pays for every argument. */
int syfi_kv_write_block(const int64_t* args);
int syfi_kv_read_block(const int64_t* args);
int syfi_paged_attention_block(const int64_t* args);

/* Synchronises `stream` and reports whether an attention kernel gave up on a bounded wait on the current device since the last
 * check (status 301; the rows that it had not finished are NaN). */
int syfi_kv_check(void* stream);

#ifdef __cplusplus
}
#endif

#endif  /* SYFI_KV_H_ */
