/*
 * cublade_kv.h - C ABI of the 8-bit paged key/value cache in
 * libcublade_quant.so: append, attention and read-back.
 *
 * No counterpart in the reference. Conventions (status codes, dtype codes,
 * streams, last-error message, workspace) are those of cublade_quant.h: raw
 * device pointers, asynchronous launches on the given stream, nothing
 * allocated, freed or synchronised.
 *
 * The cache is a pool of pages. A page holds page_size consecutive tokens of
 * one sequence; a page table row lists a sequence's pages in order. Per page
 * and kv head there is one fp32 scale for the keys and one for the values:
 *   k       [num_pages, kv_heads, page_size, head_dim]   8-bit codes
 *   v       [num_pages, kv_heads, head_dim, page_size]   8-bit codes (transposed:
 *           the attention reads 16 consecutive tokens of one dimension as one
 *           matrix-core operand, with no transposing pass)
 *   k_scale, v_scale [num_pages, kv_heads], not negative
 * A code stands for decode(code) * scale: INT8 in [-127, 127], or FP8 E4M3.
 *
 * What is on the device cannot be checked by the host, so the kernels check
 * it: a page id outside [0, num_pages) is never dereferenced. Tokens that
 * would be appended to such a page, to a page beyond the table's width or at a
 * negative position are dropped; attention over one gives NaN rows; reading
 * one back gives NaN. Two sequences that append in one call must not share the
 * page they write.
 */
#ifndef CUBLADE_KV_H
#define CUBLADE_KV_H

#include "cublade_quant.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Code types of a cache. */
enum { CBQ_KV_INT8 = 0, CBQ_KV_FP8 = 1 };

typedef struct {
  void* k;            /* 16-byte aligned */
  void* v;            /* 16-byte aligned */
  float* k_scale;
  float* v_scale;
  int64_t num_pages;  /* < 2^31 */
  int32_t kv_heads;
  int32_t head_dim;   /* a multiple of 16, 16 .. 256 */
  int32_t page_size;  /* a power of two, 16 .. 256 */
  int32_t store;      /* CBQ_KV_INT8 or CBQ_KV_FP8 */
} cbq_kv_cache;

/* The sequences of a call. lengths[b]: tokens of sequence b with the new ones.
 * cu: [batch + 1] offsets of each sequence's new tokens among the `tokens` new
 * tokens of the call, or null: one new token per sequence (tokens == batch).
 * They do not decrease. Tokens in front of cu[0] and from cu[batch] on belong to
 * no sequence (a call padded to a fixed size): they are not appended, their
 * rotated queries are NaN (as they are, without rotation; turned, with
 * positions), and their attention is that of a query that sees no key.
 * page_table: [batch, max_pages], rows table_stride elements apart. */
typedef struct {
  const int32_t* page_table;
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* cu;
  int64_t tokens;
  int32_t batch;
  int32_t max_pages;
} cbq_kv_batch;

/* One tensor of heads, [tokens, heads, head_dim] in dtype, the last dimension
 * contiguous; strides in elements, multiples of 8; data 16-byte aligned. */
typedef struct {
  const void* data;
  int64_t token_stride;
  int64_t head_stride;
} cbq_kv_heads;

/* Position rotation: pairs (x1, x2) of the first rot_dim dimensions become
 * (x1 c - x2 s, x2 c + x1 s), in fp32, every product and sum rounded. Pair i:
 * dimensions (i, i + rot_dim / 2), or (2 i, 2 i + 1) if interleaved. cos, sin:
 * [rows, rot_dim / 2] fp32, contiguous, 16-byte aligned. A token's row is its
 * index in its sequence, or positions[token] if given. rot_dim 0: no rotation.
 * A row outside [0, rows) makes the token's query NaN and its page's key
 * scale infinite (every row that attends to that page is NaN). */
typedef struct {
  const float* cos_table;
  const float* sin_table;
  const int64_t* positions;
  int64_t rows;
  int32_t rot_dim;     /* even, 0 .. head_dim */
  int32_t interleaved;
} cbq_kv_rope;

/* Appends each sequence's new keys (rotated) and values to its pages, and
 * writes its rotated queries (q.data may be null: none) to q_out
 * [tokens, q_heads, head_dim], contiguous, 16-byte aligned.
 * Scales: a page without earlier tokens gets inv = Q / max(amax, 1e-12), scale
 * = 1 / inv, codes = encode(x inv), as the quantizers of cublade_quant.h. A
 * page with earlier tokens keeps its scale if the new tokens' amax is at most
 * Q scale; else the scale is multiplied by the smallest power of two that
 * makes it so and the earlier codes are divided by it (rounded to nearest
 * even). The power of two bounds the rounding errors of repeated growth by
 * one step of the final scale. Codes behind a sequence's end keep what they
 * held. One launch. */
int cbq_kv_append(const cbq_kv_cache* cache, const cbq_kv_batch* batch, int dtype,
                  const cbq_kv_heads* k, const cbq_kv_heads* v, const cbq_kv_heads* q,
                  int32_t q_heads, const cbq_kv_rope* rope, void* q_out, cbq_stream_t stream);

/* Reads pages back: k_out, v_out [n, kv_heads, page_size, head_dim] in
 * out_dtype (CBQ_F16 / CBQ_BF16), contiguous, 16-byte aligned: T(float(code) *
 * scale). pages: n int32 page ids. A cache without pages is refused (n > 0). */
int cbq_kv_dequant(const cbq_kv_cache* cache, const int32_t* pages, int64_t n, void* k_out,
                   void* v_out, int out_dtype, cbq_stream_t stream);

/* Attention of the new tokens' queries over their sequences' cached tokens:
 *   s_j = scale * q . k_j,  o = sum_j softmax(s)_j v_j,  lse = log sum_j exp s_j
 * Query head h reads kv head h / (q_heads / kv_heads). Query i of the n of a
 * sequence of length len has position p = len - n + i and sees the keys j <= p
 * if causal, else all j < len; with window > 0 (causal only) those with
 * j > p - window. A query that sees no key gives o = 0, lse = -infinity; one
 * whose scores are all -infinity gives the NaN of their softmax, lse = -infinity.
 * Scores, statistics and sums in fp32. Probabilities are rounded to fp16 for the
 * product with the codes (not for their sum): 2^-11 of each, and 2^-25 of the
 * row's largest product of a probability and its page's value scale. bf16 queries
 * become fp16 under a power of two per row (elements below 2^-25 of the row's
 * largest vanish). Value scales that a row sees should lie within 2^100 of the
 * largest (those below 2^-64 count as 2^-64; fp16 values never lie further):
 * pages with smaller ones may be left out of the sum.
 * out: [tokens, q_heads, head_dim] in dtype, contiguous, 16-byte aligned.
 * lse: [tokens, q_heads] fp32 or null. max_length: an upper bound of lengths
 * that the host knows (0: none); only the split of the work depends on it.
 * ws: cbq_kv_attend_ws_bytes(...) bytes, 256-byte aligned (only its part
 * after the control block is used); a smaller one selects fewer splits of the
 * keys (same results within the order of fp32 sums, slower). Partial rows pass
 * through ws from one kernel of a call to the next: host threads that share a ws
 * on a stream make their calls one at a time. */
size_t cbq_kv_attend_ws_bytes(const cbq_kv_cache* cache, const cbq_kv_batch* batch,
                              int32_t q_heads, int64_t max_length);
int cbq_kv_attend(const cbq_kv_cache* cache, const cbq_kv_batch* batch, int dtype,
                  const cbq_kv_heads* q, int32_t q_heads, float scale, int causal,
                  int64_t window, int64_t max_length, void* ws, size_t ws_bytes, void* out,
                  float* lse, cbq_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* CUBLADE_KV_H */
