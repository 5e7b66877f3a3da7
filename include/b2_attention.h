/*
 * b2_attention.h -- C ABI of the cached-attention operators of
 * librdna2_b200.so: rotary positions, a paged key/value cache held in 8 bits
 * and attention over it.  Conventions as in b2_qlinear.h: int results that
 * are cudaError_t values, asynchronous work on the caller's stream,
 * caller-owned memory, no allocation and no synchronization.
 *
 * dtype codes:  0 = float32, 1 = float16, 2 = bfloat16
 * layout:       0 = half (channel i turns with i + rotary_dim / 2)
 *               1 = interleaved (channel 2i turns with 2i + 1)
 * code:         0 = int8, 1 = e4m3
 *
 * A cache is [pages][kv_heads][page][dim] codes and [pages][kv_heads] fp32
 * scales, K and V apart (page 16, 32, 64 or 128 tokens, dim 64 or 128); the
 * value of a code is code * scale.  A call serves `batch` sequences:
 * lengths[b] tokens (those of the call included), on the pages
 * table[b][0 .. width), position p on page table[b][p / page].  The call's
 * tokens are packed; sequence b has rows offsets[b] .. offsets[b + 1], or
 * tokens / batch rows each where offsets is NULL, and its last row is at
 * position lengths[b] - 1.  Table entries outside [0, pages) hold no tokens;
 * a cache of no pages needs no memory.
 */
#ifndef B2_ATTENTION_H_
#define B2_ATTENTION_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* x [tokens, heads, dim] (strides in elements, channels contiguous) -> out:
 * the first rotary_dim channels of every head rotated by the token's angles,
 * the others copied; inverse != 0 rotates back, which is also the gradient.
 * angles [angle_rows][rotary_dim] fp32: cosines, then sines; positions
 * [tokens] int32, or int64 where positions_64 != 0.  A position outside the
 * table makes NaN.  out may be x. */
int b2_rotary(const void* x, int dtype, int64_t tokens, int64_t heads, int64_t dim, int64_t x_token_stride,
              int64_t x_head_stride, const float* angles, int64_t angle_rows, int64_t rotary_dim, int layout,
              int inverse, const void* positions, int positions_64, void* out, int64_t out_token_stride,
              int64_t out_head_stride, void* stream);

/* Quantizes the call's keys (rotated where angles is given) and values
 * [tokens, kv_heads, dim] into the cache, and rotates q (may be NULL)
 * [tokens, q_heads, dim] into q_out (contiguous) in the same launch.  Rows and strides are
 * multiples of 16 bytes; rotary_dim is a multiple of 16.  For each page and
 * head that receives tokens x, with top = 127 or 448:
 *   s = max(s_old if the page holds earlier tokens, max|x| / top, 2^-100);
 *   earlier codes become RNE(code * (s_old / s)), new ones
 *   clamp(RNE(x * fp32(1 / s))).
 * No two rows of a call may fall on one page of two sequences. */
int b2_kv_append(const void* k, const void* v, int dtype, int64_t tokens, int64_t kv_heads, int64_t dim,
                 int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                 const int32_t* lengths, const int32_t* offsets, int64_t batch, const int32_t* table, int64_t width,
                 const void* q, int64_t q_heads, int64_t q_token_stride, int64_t q_head_stride, void* q_out,
                 const float* angles, int64_t angle_rows, int64_t rotary_dim, int layout, int code, void* k_codes,
                 void* v_codes, float* k_scale, float* v_scale, int64_t pages, int64_t page, void* stream);

/* Values of the n pages listed: k_out, v_out [n][kv_heads][page][dim], and
 * their scales [2][n][kv_heads] (keys, then values) where scales_out is given;
 * NaN for a page outside the cache. */
int b2_kv_read(const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale, int code,
               int64_t num_pages, int64_t kv_heads, int64_t page, int64_t dim, const int32_t* pages, int64_t n,
               int dtype, void* k_out, void* v_out, float* scales_out, void* stream);

/* Attention of q [tokens, q_heads, dim] (fp16 or bf16) over the cache; query
 * head h reads kv head h / (q_heads / kv_heads).  A row at position p sees
 * the cached tokens j < lengths[b], with causal != 0 only j <= p, with
 * window > 0 only j > p - window.  out [tokens, q_heads, dim] in q's dtype
 * and, where lse is given, the natural logarithm of each row's sum of
 * exponentials [tokens, q_heads]; a row that sees nothing gives zeros and
 * -inf.  Scales are not negative, value scales below 2^-100 count as 2^-100,
 * and e4m3 codes before a sequence's end are no NaN; a scale that is NaN or
 * infinite makes NaN of the rows that see its block, and of no others.
 * max_new bounds the tokens of one sequence.  The workspace holds
 * b2_kv_attention_workspace_bytes bytes, 256-byte aligned, zero-filled
 * before its first call; every call leaves it ready for the next one on the
 * same stream, of any shape that it is large enough for. */
size_t b2_kv_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t max_new, int64_t q_heads,
                                       int64_t kv_heads, int64_t dim, int64_t width, int64_t page, int64_t window);
int b2_kv_attention(const void* q, int dtype, int64_t tokens, int64_t q_heads, int64_t q_token_stride,
                    int64_t q_head_stride, const int32_t* lengths, const int32_t* offsets, int64_t batch,
                    int64_t max_new, const int32_t* table, int64_t width, int code, const void* k_codes,
                    const void* v_codes, const float* k_scale, const float* v_scale, int64_t pages, int64_t kv_heads,
                    int64_t page, int64_t dim, float scale, int causal, int64_t window, void* out, float* lse,
                    void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* B2_ATTENTION_H_ */
