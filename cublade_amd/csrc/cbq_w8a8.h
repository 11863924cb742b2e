// cbq_w8a8.h - what the kernels of the INT8 x INT8 products share: their
// arguments, the activations, and the step from an integer sum to an output.
#pragma once

#include "cbq_device.h"
#include "cbq_host.h"
#include "cublade_w8a8.h"

namespace cbq {

typedef int i4v __attribute__((ext_vector_type(4)));
typedef int i16x __attribute__((ext_vector_type(16)));
typedef float f4v __attribute__((ext_vector_type(4)));

// Activation of the gate; kNoAct: a single product (linear).
enum : int { kNoAct = -1 };

struct W8Args {
  const uint8_t* x;        // [M] rows of K codes, ldx bytes apart
  const uint8_t* w[2];     // [N] rows of K codes (gated: the gate's, the up projection's)
  int64_t ldx, ldw[2];
  const float* sx;         // scales: sx[m sx_step], sw[p][n sw_step[p]]
  const float* sw[2];
  int64_t sx_step, sw_step[2];
  const void* bias[2];     // [N] in bias_dt, or null
  int bias_dt;
  int act;
  void* y;                 // [M, N] in out_dt
  int out_dt;
  int vec;                 // y's rows may be stored 16 bytes at a time
  int M, N, K;
  int tiles_m, tiles_n;
  int splits, split_steps; // K in ranges of split_steps 128-byte steps
  int* part;               // sums of the ranges: [splits][tiles], as the tiles' registers hold them
};

// act(g) in fp32. The sigmoids take the hardware's 2^x and reciprocal (1 ulp
// each); the argument's rounding costs |g| 2^-24 of e^-g. 
__device__ __forceinline__ float sigmoid_of(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}

template <int ACT>
__device__ __forceinline__ float activate(float g) {
  if constexpr (ACT == CBQ_ACT_SILU) return g * sigmoid_of(g);
  // 1/2 (1 + tanh(u)) = sigmoid(2 u)
  else if constexpr (ACT == CBQ_ACT_GELU_TANH)
    return g * sigmoid_of(g * (1.59576912f + 0.0713548163f * (g * g)));
  // 1 + erf(t) = erfc(-t), which keeps its digits where g is negative
  else if constexpr (ACT == CBQ_ACT_GELU) return 0.5f * g * erfcf(g * -0.707106781f);
  else if constexpr (ACT == CBQ_ACT_RELU) return g < 0.0f ? 0.0f : g;
  else return g;
}

// The same for an activation known at run time (the same for all threads).
__device__ __forceinline__ float activate(int act, float g) {
  switch (act) {
    case CBQ_ACT_SILU: return activate<CBQ_ACT_SILU>(g);
    case CBQ_ACT_GELU: return activate<CBQ_ACT_GELU>(g);
    case CBQ_ACT_GELU_TANH: return activate<CBQ_ACT_GELU_TANH>(g);
    default: return activate<CBQ_ACT_RELU>(g);
  }
}

__device__ __forceinline__ float ld_any(const void* p, int dt, int64_t i) {
  return dt == kF32 ? ld1<kF32>(p, i) : dt == kF16 ? ld1<kF16>(p, i) : ld1<kBF16>(p, i);
}

// 16 bytes of a row of K >= 16 codes at min(k, K - 16), at any address.
__device__ __forceinline__ u32x4 ld_codes(const uint8_t* row, int k, int K) {
  typedef u32x4 __attribute__((aligned(1))) u32x4_any;
  return *reinterpret_cast<const u32x4_any*>(row + min(k, K - 16));
}

// The codes k .. k + 15 of what ld_codes loaded for them, with zeros from K on.
__device__ __forceinline__ u32x4 from_k(u32x4 v, int k, int K) {
  if (const int d = k - min(k, K - 16)) {   // the row's last chunk: moved down
    if (d & 8) v = u32x4{v.z, v.w, 0u, 0u};
    if (d & 4) v = u32x4{v.y, v.z, v.w, 0u};
    v = u32x4{__builtin_amdgcn_alignbyte(v.y, v.x, d & 3), __builtin_amdgcn_alignbyte(v.z, v.y, d & 3),
              __builtin_amdgcn_alignbyte(v.w, v.z, d & 3), __builtin_amdgcn_alignbyte(0u, v.w, d & 3)};
    if (d >= 16) v = u32x4{0u, 0u, 0u, 0u};
  }
  return v;
}

// An integer sum with its scales and bias.
__device__ __forceinline__ float scaled(int sum, float sx, float sw, float b) {
  return static_cast<float>(sum) * sx * sw + b;
}

__device__ __forceinline__ void st_any(void* y, int dt, int64_t i, float v) {
  if (dt == kF32) static_cast<float*>(y)[i] = v;
  else if (dt == kF16) static_cast<uint16_t*>(y)[i] = out1<kF16>(v);
  else static_cast<uint16_t*>(y)[i] = out1<kBF16>(v);
}

// Four neighbouring outputs y[m, n .. n + 3] (n % 4 == 0).
__device__ __forceinline__ void st_quad(const W8Args& a, int64_t m, int n, f4v v) {
  const int64_t i = m * a.N + n;
  if (a.vec && n + 3 < a.N) {
    if (a.out_dt == kF32) *reinterpret_cast<f4v*>(static_cast<float*>(a.y) + i) = v;
    else
      *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.y) + i) =
          a.out_dt == kF16 ? u32x2{pack2_out<kF16>(v.x, v.y), pack2_out<kF16>(v.z, v.w)}
                           : u32x2{pack2_out<kBF16>(v.x, v.y), pack2_out<kBF16>(v.z, v.w)};
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (n + q < a.N) st_any(a.y, a.out_dt, i + q, v[q]);
  }
}

// Calls f with the activation as a constant.
template <typename F>
inline void with_act(int act, F&& f) {
  switch (act) {
    case CBQ_ACT_SILU: f(std::integral_constant<int, CBQ_ACT_SILU>{}); break;
    case CBQ_ACT_GELU: f(std::integral_constant<int, CBQ_ACT_GELU>{}); break;
    case CBQ_ACT_GELU_TANH: f(std::integral_constant<int, CBQ_ACT_GELU_TANH>{}); break;
    case CBQ_ACT_RELU: f(std::integral_constant<int, CBQ_ACT_RELU>{}); break;
    default: f(std::integral_constant<int, kNoAct>{}); break;
  }
}

// What rows of codes and their strides are multiples of.
enum { kRows16, kRows4, kRows1 };

// cbq_w8a8_few.hip: few rows of x, or few outputs; K >= 16. The shape for these sizes (-1:
// none) and its modelled time; any: rows that are no multiples of 16 bytes. Returns after queueing.
// The model was fitted up to 1024 rows; past kFewRows only tiles are considered.
constexpr int kFewRows = 2048;
struct FewPlan { int shape; double us; };
FewPlan few_plan(int64_t M, int64_t N, int64_t K, int proj, int rows, int cus);
void launch_w8a8_few(const W8Args& a, int shape, bool any, hipStream_t s);
cbq_w8a8_form few_form(int shape, int64_t M, int64_t N, int proj, int rows);

}  // namespace cbq
