/*
 * cublade_w8a8.h - C ABI of the products of INT8 activations and INT8 weights
 * and of the norms around a block, in libcublade_quant.so.
 *
 * No counterpart in the reference. Conventions (status codes, dtype codes,
 * streams, last-error message, workspace) are those of cublade_quant.h: raw
 * device pointers, asynchronous launches on the given stream, nothing
 * allocated, freed or synchronised.
 */
#ifndef CUBLADE_W8A8_H
#define CUBLADE_W8A8_H

#include "cublade_quant.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rows of INT8 codes, `stride` bytes apart: row r's element k stands for
 * data[r stride + k] scale[r scale_stride]; scale_stride 1: a scale for each
 * row (token, output channel), 0: one for all. */
typedef struct {
  const int8_t* data;
  int64_t stride;
  const float* scale;
  int64_t scale_stride;
} cbq_i8_rows;

/* Activations: codes of x's rows (tokens) with a scale for each, by the kernels and with the
 * workspace of cbq_quant_int8_channel (axis 0) and the same bits, but for rows that hold a NaN
 * or an infinity: those get a NaN scale (and codes 0), so that a product's row is NaN. There,
 * NaN inputs are left out of the maximum, as in the reference. */
int cbq_quant_int8_tokens(const void* x, int dtype, int64_t rows, int64_t cols, float eps,
                          void* ws, size_t ws_bytes, int8_t* q, float* scale,
                          cbq_stream_t stream);

/* Activations of the gated product. GELU: with the error function, or its
 * approximation by tanh. */
enum { CBQ_ACT_SILU = 0, CBQ_ACT_GELU = 1, CBQ_ACT_GELU_TANH = 2, CBQ_ACT_RELU = 3 };

/* y[m, n] = sx[m] sw[n] (sum_k x[m, k] w[n, k]) + bias[n]
 * x: M rows, w: N rows, of K codes (strides up to 2^22); K <= 131071, so that the int32 sums are
 * exact for any codes. y: [M, N] in out_dtype, contiguous. bias (or null): [N]
 * in bias_dtype. The sum becomes fp32 (rounded once past 2^24), the rest is
 * fp32 with each product and sum rounded, then one rounding to out_dtype.
 * A launch takes fewer than 2^32 threads, so K < 16 takes M N below 2^32 - 256, and others
 * fewer than 2^24 tiles of 256 x 256.
 *
 * ws: cbq_w8a8_ws_bytes(M, N, K, 1) bytes, 256-byte aligned, of which the
 * control block is not used. With less, or none, K is not cut into ranges, and
 * rows that are no multiples of 16 bytes are not copied to such (same results,
 * slower). Sums and copies pass through ws from one kernel of a call to the next:
 * host threads that share a ws on a stream make their calls one at a time.
 * Codes may have any alignment; x and w, their strides and K in multiples of 16
 * bytes are faster. */
size_t cbq_w8a8_ws_bytes(int64_t M, int64_t N, int64_t K, int projections);
int cbq_w8a8_linear(const cbq_i8_rows* x, const cbq_i8_rows* w, const void* bias, int bias_dtype,
                    int64_t M, int64_t N, int64_t K, void* y, int out_dtype, void* ws,
                    size_t ws_bytes, cbq_stream_t stream);

/* y[m, n] = act(g) u, with g and u the products above of the same x with the
 * rows of `gate` and of `up` (each bias may be null; both have bias_dtype). ws:
 * cbq_w8a8_ws_bytes(M, N, K, 2). */
int cbq_w8a8_gated(const cbq_i8_rows* x, const cbq_i8_rows* gate, const cbq_i8_rows* up,
                   const void* gate_bias, const void* up_bias, int bias_dtype, int activation,
                   int64_t M, int64_t N, int64_t K, void* y, int out_dtype, void* ws,
                   size_t ws_bytes, cbq_stream_t stream);

/* How a product of these sizes is computed (projections as above), for tests and tuning; nothing
 * is launched. multiple: what the rows of all operands are multiples of (address, stride and K,
 * in bytes): 16, 4 or 1. With the workspace that cbq_w8a8_ws_bytes names. */
enum { CBQ_W8A8_SHORT = 0, CBQ_W8A8_FEW = 1, CBQ_W8A8_TILES = 2 };

typedef struct {
  int32_t kernel;
  int32_t weight_rows, x_rows;   /* that a workgroup owns (weight rows: of all projections) */
  int32_t threads;               /* of a workgroup */
  int32_t stages;                /* in LDS, of a wave (FEW) or a workgroup (TILES) */
  int32_t ranges;                /* of K, each with workgroups of its own */
  int32_t copies;                /* 1: x and the weights are copied to rows of whole 16 bytes */
  int64_t workgroups;
} cbq_w8a8_form;

int cbq_w8a8_form_of(int64_t M, int64_t N, int64_t K, int projections, int multiple,
                     cbq_w8a8_form* form);

/* The norms before and after a block, with the block's gate and residual scale:
 *   t = post ? norm(x; post_weight, post_bias) : x
 *   h = residual + alpha gate t            (rounded to the residual's type)
 *   n = norm(h; weight, bias)              (without a residual: of x)
 * norm(v) = (v - mean) / sqrt(var + eps) weight + bias over a token's `hidden`
 * elements; CBQ_NORM_RMS: mean = 0. A null weight is 1, a null bias 0, a null
 * gate 1. out_dtype CBQ_I8: codes of n and a scale for each token, as by
 * cbq_quant_int8_channel (axis 0) of n in fp32; a token with a NaN or an
 * infinity, in x or in n, gets a NaN scale. Otherwise n in out_dtype. out null: h only.
 *
 * x: [tokens, hidden], rows x_stride elements apart, in x_dtype. residual (or
 * null): likewise, in x's type or CBQ_F32. h: [tokens, hidden] in the residual's
 * type, contiguous. Parameters: [hidden] in param_dtype. gate: element (t, c) at
 * gate[t gate_token_stride + c gate_channel_stride]. out: contiguous. scale:
 * [tokens]. Every tensor is aligned to its elements. h and out do not overlap
 * what is read. All in fp32: sums of squares overflow (n = 0) where a token's
 * elements pass about 2^63. One launch for each 2^21 tokens. */
enum { CBQ_NORM_RMS = 0, CBQ_NORM_LAYER = 1 };

typedef struct {
  int64_t tokens, hidden;
  const void* x;
  int64_t x_stride;
  const void* residual;
  int64_t residual_stride;
  const void* gate;
  int64_t gate_token_stride, gate_channel_stride;
  const void* post_weight;
  const void* post_bias;
  const void* weight;
  const void* bias;
  void* h;
  void* out;
  float* scale;
  int32_t x_dtype, residual_dtype, param_dtype, gate_dtype, out_dtype;
  int32_t kind, post;
  float eps, alpha;
} cbq_norm_args;

int cbq_norm(const cbq_norm_args* args, cbq_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* CUBLADE_W8A8_H */
