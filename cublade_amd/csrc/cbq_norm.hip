// cbq_norm.hip - the norms before and after a block, with the block's gate and
// residual scale; the result leaves as INT8 codes with a scale for each token (the
// activations of the INT8 products), or as floating-point values.
//
//   t = post ? norm(x) : x          norm(v) = (v - mean) rstd weight + bias
//   h = residual + alpha gate t     (rounded to the residual's type and stored)
//   n = norm(h)                     (without a residual: norm(x))
//   inv = 127 / max(max |n|, 1e-12), scale = 1 / inv, codes = rne(n inv)
//
// rms: mean = 0; rstd = 1 / sqrt(sum (v - mean)^2 / hidden + eps). All of it in fp32.
// n is the norm of h as stored, so that it is what a later call would find.
//
// A row is held in registers from its loads to its last store: each tensor is read
// and written once. What bounds the kernel is
// memory for many tokens, and the chain of load, reductions and store for few.
// The sum of squares and the largest |v weight| are reduced together: rounding is
// monotonic, so max |v weight| rstd is the largest of the rounded products.
//
// A NaN or an infinity in a row makes its maximum NaN (maxima are taken over the bit
// patterns of absolute values, where a NaN is above everything) and with it the scale, as
// does a norm that is infinite itself (a weight, a bias, a product past fp32):
// the token's outputs of a product are NaN rather than those of zero codes.
#include <algorithm>
#include <type_traits>

#include "cbq_device.h"
#include "cbq_host.h"
#include "cublade_w8a8.h"

namespace cbq {
namespace {

typedef u32x4 __attribute__((aligned(4))) u32x4_a4;
typedef u32x2 __attribute__((aligned(4))) u32x2_a4;

// A thread holds 8 V elements of its row, of nt threads. Even rows (whole chunks of 8,
// every tensor's rows on multiples of 4 bytes): the chunks t, t + nt, ..., a load of 16
// bytes each. Odd rows: the elements t, t + nt, ..., one by one; vector loads that are
// not on a multiple of 4 pass the address unit lane by lane, and a row's partial chunk
// element by element takes more instructions than the rest of the row.
// 32-bit indices, rows at addresses the wave has in common: a load or store is then one
// instruction with its offset in a register.
template <bool ODD>
__device__ __forceinline__ uint32_t index_of(int t, int nt, int v, int k) {
  return ODD ? t + (8 * v + k) * nt : (t + v * nt) * 8 + k;
}

// Eight elements as loaded: even rows' words (16-bit types: the first 4), or an odd
// row's elements.
struct Raw { uint32_t w[8]; };

template <int DT, bool ODD, bool CLAMP, bool NT = false>
__device__ __forceinline__ Raw ld_raw(const void* row, int t, int nt, int v, uint32_t H) {
  Raw r = {};
  if constexpr (ODD) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t e = index_of<true>(t, nt, v, k);
      if (CLAMP || e < H) {
        const uint32_t c = CLAMP ? min(e, H - 1) : e;
        if constexpr (DT == kF32) r.w[k] = static_cast<const uint32_t*>(row)[c];
        else r.w[k] = static_cast<const uint16_t*>(row)[c];
      }
    }
  } else if (index_of<false>(t, nt, v, 0) < H) {
    const char* p = static_cast<const char*>(row) + index_of<false>(t, nt, v, 0) * elem_bytes<DT>();
#pragma unroll
    for (int h = 0; h < (DT == kF32 ? 2 : 1); ++h) {
      const u32x4_a4* q = reinterpret_cast<const u32x4_a4*>(p + 16 * h);
      const u32x4 x = NT ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[4 * h + i] = x[i];
    }
  }
  return r;
}

template <int DT, bool ODD>
__device__ __forceinline__ void widen(const Raw& r, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (DT == kF32) {
      f[k] = __uint_as_float(r.w[k]);
    } else {
      const uint32_t w = ODD ? r.w[k] : r.w[k >> 1];
      const f32x2 p = pair_to_f32<DT>(w);
      f[k] = !ODD && (k & 1) ? p.y : p.x;
    }
  }
}

// The same for a type known at run time only (the same for all threads).
template <bool ODD, bool CLAMP>
__device__ __forceinline__ Raw ld_raw(const void* row, int dt, int t, int nt, int v, uint32_t H) {
  return dt == kF32 ? ld_raw<kF32, ODD, CLAMP>(row, t, nt, v, H) : ld_raw<kF16, ODD, CLAMP>(row, t, nt, v, H);
}
template <bool ODD>
__device__ __forceinline__ void widen(const Raw& r, int dt, float (&f)[8]) {
  if (dt == kF32) widen<kF32, ODD>(r, f);
  else if (dt == kF16) widen<kF16, ODD>(r, f);
  else widen<kBF16, ODD>(r, f);
}

// f rounded to DT, as ld_raw would load it.
template <int DT, bool ODD>
__device__ __forceinline__ Raw narrow(const float (&f)[8]) {
  Raw r = {};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (DT == kF32) r.w[k] = __float_as_uint(f[k]);
    else if constexpr (ODD) r.w[k] = pack2_out<DT>(f[k], 0.0f) & 0xffffu;
    else if (k % 2 == 0) r.w[k >> 1] = pack2_out<DT>(f[k], f[k + 1]);
  }
  return r;
}

template <int DT, bool ODD>
__device__ __forceinline__ void st_raw(void* row, int t, int nt, int v, uint32_t H, const Raw& r) {
  if constexpr (ODD) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t e = index_of<true>(t, nt, v, k);
      if (e < H) {
        if constexpr (DT == kF32) static_cast<uint32_t*>(row)[e] = r.w[k];
        else static_cast<uint16_t*>(row)[e] = static_cast<uint16_t>(r.w[k]);
      }
    }
  } else if (index_of<false>(t, nt, v, 0) < H) {
    char* p = static_cast<char*>(row) + index_of<false>(t, nt, v, 0) * elem_bytes<DT>();
#pragma unroll
    for (int h = 0; h < (DT == kF32 ? 2 : 1); ++h)
      *reinterpret_cast<u32x4_a4*>(p + 16 * h) = u32x4{r.w[4 * h], r.w[4 * h + 1], r.w[4 * h + 2], r.w[4 * h + 3]};
  }
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Sums and maxima over a row's threads; every thread gets them. Within a wave by DPP
// (a reduction by shuffles through LDS takes 6 round trips of its latency): neighbours,
// quads and rows of 16 by permutations that every lane takes part in, then the rows'
// results handed on to lane 63.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {   // 0 where no lane is handed on
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false));
}

template <typename F>
__device__ __forceinline__ uint32_t wave_fold(uint32_t v, F&& f) {
  v = f(v, dpp_u32<0xB1, 0xF>(v));    // quad_perm [1,0,3,2]
  v = f(v, dpp_u32<0x4E, 0xF>(v));    // quad_perm [2,3,0,1]
  v = f(v, dpp_u32<0x141, 0xF>(v));   // row_half_mirror
  v = f(v, dpp_u32<0x140, 0xF>(v));   // row_mirror
  v = f(v, dpp_u32<0x142, 0xA>(v));   // row_bcast15, to rows 1 and 3
  v = f(v, dpp_u32<0x143, 0xC>(v));   // row_bcast31, to rows 2 and 3
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), kWave - 1));
}

__device__ __forceinline__ uint32_t add_f32(uint32_t a, uint32_t b) {
  return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}
__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }

constexpr int kMaxWaves = 16;

// slots: a set for each reduction of the kernel.
template <bool WAVE>
__device__ __forceinline__ float row_sum(float sum, uint32_t* slots) {
  uint32_t s = wave_fold(__float_as_uint(sum), add_f32);
  if constexpr (!WAVE) {
    if (threadIdx.x % kWave == 0) slots[threadIdx.x / kWave] = s;
    __syncthreads();
    s = slots[0];
    for (int w = 1; w < static_cast<int>(blockDim.x) / kWave; ++w) s = add_f32(s, slots[w]);
  }
  return __uint_as_float(s);
}

struct Stat { float sum; uint32_t top; };

template <bool WAVE>
__device__ __forceinline__ Stat row_stat(Stat v, uint32_t* slots) {
  uint32_t s = wave_fold(__float_as_uint(v.sum), add_f32), t = wave_fold(v.top, max_u32);
  if constexpr (!WAVE) {
    if (threadIdx.x % kWave == 0) {
      slots[threadIdx.x / kWave] = s;
      slots[kMaxWaves + threadIdx.x / kWave] = t;
    }
    __syncthreads();
    s = slots[0];
    t = slots[kMaxWaves];
    for (int w = 1; w < static_cast<int>(blockDim.x) / kWave; ++w) {
      s = add_f32(s, slots[w]);
      t = max_u32(t, slots[kMaxWaves + w]);
    }
  }
  return {__uint_as_float(s), t};
}

constexpr float kEps = 1e-12f;   // of a row's maximum, as in the quantizers

struct Norm {
  int layer;               // else rms
  float eps;
  float inv_h;
};

__device__ __forceinline__ float rstd_of(float ss, const Norm& n) {
  return rsqrtf(ss * n.inv_h + n.eps);   // eps may be 0, and v_rsq_f32 takes no denormals
}

struct Args {
  cbq_norm_args a;
  Norm n;
  int stream;              // x and the residual are loaded past the caches
};

template <bool ODD>
__device__ __forceinline__ void st_out(const cbq_norm_args& a, int64_t token, int t, int nt, int v,
                                       const float (&f)[8], float inv) {
  const uint32_t H = static_cast<uint32_t>(a.hidden);
  if (a.out_dtype == CBQ_I8) {
    uint8_t* row = static_cast<uint8_t*>(a.out) + token * a.hidden;
    if constexpr (ODD) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t e = index_of<true>(t, nt, v, k);
        if (e < H) row[e] = static_cast<uint8_t>(q_int8(f[k] * inv));
      }
    } else if (index_of<false>(t, nt, v, 0) < H) {
      const uint2 q = pack8_int8(f, inv);
      *reinterpret_cast<u32x2_a4*>(row + index_of<false>(t, nt, v, 0)) = u32x2{q.x, q.y};
    }
    return;
  }
  char* row = static_cast<char*>(a.out) + token * a.hidden * (a.out_dtype == CBQ_F32 ? 4 : 2);
  if (a.out_dtype == CBQ_F32) st_raw<kF32, ODD>(row, t, nt, v, H, narrow<kF32, ODD>(f));
  else if (a.out_dtype == CBQ_F16) st_raw<kF16, ODD>(row, t, nt, v, H, narrow<kF16, ODD>(f));
  else st_raw<kBF16, ODD>(row, t, nt, v, H, narrow<kBF16, ODD>(f));
}

// Row `token` of the gate, or the values it repeats.
__device__ __forceinline__ const char* gate_row(const cbq_norm_args& a, int64_t token) {
  return static_cast<const char*>(a.gate) + token * a.gate_token_stride * (a.gate_dtype == CBQ_F32 ? 4 : 2);
}

template <int DT>
__device__ __forceinline__ const char* row_of(const void* p, int64_t token, int64_t stride) {
  return static_cast<const char*>(p) + token * stride * elem_bytes<DT>();
}

// WAVE: a row per wave, 4 to a workgroup; else a row per workgroup of any number of
// waves.
template <int XT, int RT, int V, bool WAVE, bool ODD>
__global__ __launch_bounds__(WAVE ? kBlock : 1024) void k_norm(Args args) {
  const cbq_norm_args& a = args.a;
  __shared__ uint32_t slots[5][2 * kMaxWaves];
  const uint32_t H = static_cast<uint32_t>(a.hidden);
  const int64_t token = WAVE ? blockIdx.x * (kBlock / kWave) +
                                   __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave)
                             : blockIdx.x;
  if (WAVE && token >= a.tokens) return;
  const int t = WAVE ? threadIdx.x % kWave : threadIdx.x;
  const int nt = WAVE ? kWave : blockDim.x;

  // All of the row's loads first. Odd rows, one element at a time: loads past the row's end
  // take the last element again, whose value is not used, since a load under a condition
  // waits for the one before (3001 x 1403: 15.4 -> 13.9 us); not with two chunks, whose
  // loads would all need registers at once.
  constexpr bool CLAMP = V == 1;
  Raw rx[V], rr[V], rw[V];
  auto loads = [&](auto stream) {
    constexpr bool NT = decltype(stream)::value;
#pragma unroll
    for (int v = 0; v < V; ++v)
      rx[v] = ld_raw<XT, ODD, CLAMP, NT>(row_of<XT>(a.x, token, a.x_stride), t, nt, v, H);
    if (a.residual) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        rr[v] = ld_raw<RT, ODD, CLAMP, NT>(row_of<RT>(a.residual, token, a.residual_stride), t, nt, v, H);
    }
  };
  if (args.stream) loads(std::true_type{});
  else loads(std::false_type{});
  constexpr bool HELD = V <= 2 && !ODD;   // else no registers to spare
  if (HELD && a.weight) {
#pragma unroll
    for (int v = 0; v < V; ++v) rw[v] = ld_raw<ODD, CLAMP>(a.weight, a.param_dtype, t, nt, v, H);
  }
  float f[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v) widen<XT, ODD>(rx[v], f[v]);

  auto each = [&](auto&& fn) {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < 8; ++k) fn(v, k);
  };
  auto inside = [&](int v, int k) { return index_of<ODD>(t, nt, v, ODD ? k : 0) < H; };
  if constexpr (ODD && CLAMP) each([&](int v, int k) { f[v][k] = inside(v, k) ? f[v][k] : 0.0f; });
  // layer: the mean leaves f. Elements past the row stay zero.
  auto centre = [&](uint32_t* s) {
    if (!args.n.layer) return;
    float sum = 0.0f;
    each([&](int v, int k) { sum += f[v][k]; });
    const float mean = row_sum<WAVE>(sum, s) * args.n.inv_h;
    each([&](int v, int k) { f[v][k] = inside(v, k) ? f[v][k] - mean : 0.0f; });
  };
  auto squares = [&] {
    float ss = 0.0f;
    each([&](int v, int k) { ss += f[v][k] * f[v][k]; });
    return ss;
  };
  // f = f p, or f + p, with a parameter of the channels.
  auto with_param = [&](const void* p, int dt, const Raw* held, auto&& op) {
    if (!p) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float w[8];
      widen<ODD>(held ? held[v] : ld_raw<ODD, CLAMP>(p, dt, t, nt, v, H), dt, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[v][k] = op(f[v][k], w[k]);
    }
  };
  auto times = [](float x, float y) { return x * y; };
  auto plus = [](float x, float y) { return x + y; };

  if (a.residual) {
    if (a.post) {
      centre(slots[0]);
      const float rstd = rstd_of(row_sum<WAVE>(squares(), slots[1]), args.n);
      with_param(a.post_weight, a.param_dtype, nullptr, times);
      each([&](int v, int k) { f[v][k] *= rstd; });
      with_param(a.post_bias, a.param_dtype, nullptr, plus);
    }
    if (a.gate) {
      const char* g = gate_row(a, token);
      if (a.gate_channel_stride == 0) {
        const float gv = a.gate_dtype == CBQ_F32 ? ld1<kF32>(g, 0)
                         : a.gate_dtype == CBQ_F16 ? ld1<kF16>(g, 0) : ld1<kBF16>(g, 0);
        each([&](int v, int k) { f[v][k] *= gv; });
      } else {
        with_param(g, a.gate_dtype, nullptr, times);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float r[8];
      widen<RT, ODD>(rr[v], r);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[v][k] = r[k] + a.alpha * f[v][k];
      const Raw o = narrow<RT, ODD>(f[v]);
      st_raw<RT, ODD>(static_cast<char*>(a.h) + token * a.hidden * elem_bytes<RT>(), t, nt, v, H, o);
      widen<RT, ODD>(o, f[v]);
    }
    each([&](int v, int k) { f[v][k] = inside(v, k) ? f[v][k] : 0.0f; });
  }
  if (!a.out) return;

  centre(slots[2]);
  Stat s = {squares(), 0u};
  with_param(a.weight, a.param_dtype, HELD ? rw : nullptr, times);
  each([&](int v, int k) { s.top = max_u32(s.top, abs_bits(f[v][k])); });
  s = row_stat<WAVE>(s, slots[3]);
  const float rstd = rstd_of(s.sum, args.n);
  each([&](int v, int k) { f[v][k] *= rstd; });
  float amax = __uint_as_float(s.top) * rstd, inv = 0.0f;
  if (a.bias) {
    with_param(a.bias, a.param_dtype, nullptr, plus);
    if (a.out_dtype == CBQ_I8) {
      uint32_t top = 0u;
      each([&](int v, int k) { top = inside(v, k) ? max_u32(top, abs_bits(f[v][k])) : top; });
      amax = __uint_as_float(row_stat<WAVE>({0.0f, top}, slots[4]).top);
    }
  }
  if (a.out_dtype == CBQ_I8) {
    inv = row_inv<true>(amax, kEps);
    if (t == 0) a.scale[token] = 1.0f / inv;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) st_out<ODD>(a, token, t, nt, v, f[v], inv);
}

// Rows too long for registers: a workgroup of 1024 per row, which reads its row again
// for each sum (h from where this thread stored it), element by element.
template <int XT, int RT>
__global__ __launch_bounds__(1024) void k_norm_long(Args args) {
  const cbq_norm_args& a = args.a;
  __shared__ uint32_t slots[5][2 * kMaxWaves];
  const int64_t H = a.hidden, token = blockIdx.x;
  const char* x = row_of<XT>(a.x, token, a.x_stride);
  const char* r = row_of<RT>(a.residual, token, a.residual_stride);
  char* h = static_cast<char*>(a.h) + (a.residual ? token * H * elem_bytes<RT>() : 0);
  const char* g = a.gate ? gate_row(a, token) : nullptr;
  auto each = [&](auto&& fn) {
    for (int64_t e = threadIdx.x; e < H; e += 1024) fn(e);
  };
  auto ld_p = [&](const void* p, int dt, int64_t e) {
    return dt == kF32 ? ld1<kF32>(p, e) : dt == kF16 ? ld1<kF16>(p, e) : ld1<kBF16>(p, e);
  };
  auto ld_x = [&](int64_t e) { return ld1<XT>(x, e); };
  auto ld_v = [&](int64_t e) { return a.residual ? ld1<RT>(h, e) : ld1<XT>(x, e); };   // what the last norm is of
  auto moments = [&](auto&& ld, uint32_t* s0, uint32_t* s1, float& mean) {
    mean = 0.0f;
    if (args.n.layer) {
      float sum = 0.0f;
      each([&](int64_t e) { sum += ld(e); });
      mean = row_sum<false>(sum, s0) * args.n.inv_h;
    }
    float ss = 0.0f;
    each([&](int64_t e) {
      const float d = ld(e) - mean;
      ss += d * d;
    });
    return rstd_of(row_sum<false>(ss, s1), args.n);
  };
  auto normed = [&](float v, int64_t e, float mean, float rstd, const void* w, const void* b) {
    v -= mean;
    if (w) v *= ld_p(w, a.param_dtype, e);
    v *= rstd;
    return b ? v + ld_p(b, a.param_dtype, e) : v;
  };
  float mean = 0.0f, rstd = 1.0f;
  if (a.residual) {
    if (a.post) rstd = moments(ld_x, slots[0], slots[1], mean);
    each([&](int64_t e) {
      float v = ld_x(e);
      if (a.post) v = normed(v, e, mean, rstd, a.post_weight, a.post_bias);
      if (g) v *= ld_p(g, a.gate_dtype, e * a.gate_channel_stride);
      v = ld1<RT>(r, e) + a.alpha * v;
      if constexpr (RT == kF32) reinterpret_cast<float*>(h)[e] = v;
      else reinterpret_cast<uint16_t*>(h)[e] = out1<RT>(v);
    });
  }
  if (!a.out) return;
  rstd = moments(ld_v, slots[2], slots[3], mean);
  float inv = 0.0f;
  if (a.out_dtype == CBQ_I8) {
    uint32_t top = 0u;
    each([&](int64_t e) { top = max_u32(top, abs_bits(normed(ld_v(e), e, mean, rstd, a.weight, a.bias))); });
    inv = row_inv<true>(__uint_as_float(row_stat<false>({0.0f, top}, slots[4]).top), kEps);
    if (threadIdx.x == 0) a.scale[token] = 1.0f / inv;
  }
  each([&](int64_t e) {
    const float v = normed(ld_v(e), e, mean, rstd, a.weight, a.bias);
    const int64_t i = token * H + e;
    if (a.out_dtype == CBQ_I8) static_cast<uint8_t*>(a.out)[i] = static_cast<uint8_t>(q_int8(v * inv));
    else if (a.out_dtype == CBQ_F32) static_cast<float*>(a.out)[i] = v;
    else static_cast<uint16_t*>(a.out)[i] = a.out_dtype == CBQ_F16 ? out1<kF16>(v) : out1<kBF16>(v);
  });
}

template <int XT, int RT, bool ODD>
void launch_rows(const Args& args, hipStream_t s) {
  const int64_t chunks = cdiv(args.a.hidden, 8), tokens = args.a.tokens;
  const unsigned rows = static_cast<unsigned>(tokens);
  const unsigned quads = static_cast<unsigned>(cdiv(tokens, kBlock / kWave));
  auto threads = [](int64_t per) { return static_cast<unsigned>(cdiv(per, kWave) * kWave); };
  // One chunk per thread for few tokens, where the chain of a row counts; two for
  // many, where more rows in flight and fewer reductions do (16384 x 1152, one / two:
  // 26.9 / 24.4 us, 16384 x 1408 29.7 / 28.0), but for odd rows from 4096 elements on
  // (4096 x 2049: 15.6 / 16.3, 4096 x 8001 54 / 51).
  const bool many = tokens > 2 * device_cus();
  if (chunks <= kWave) k_norm<XT, RT, 1, true, ODD><<<quads, kBlock, 0, s>>>(args);
  else if (chunks <= 2 * kWave) k_norm<XT, RT, 2, true, ODD><<<quads, kBlock, 0, s>>>(args);
  else if (chunks <= 1024 && !(many && chunks > (ODD ? 512 : 128)))
    k_norm<XT, RT, 1, false, ODD><<<rows, threads(chunks), 0, s>>>(args);
  else if (chunks <= 2048) k_norm<XT, RT, 2, false, ODD><<<rows, threads(cdiv(chunks, 2)), 0, s>>>(args);
  else if (!ODD && chunks <= 4096) k_norm<XT, RT, 4, false, false><<<rows, threads(cdiv(chunks, 4)), 0, s>>>(args);
  else k_norm_long<XT, RT><<<rows, 1024, 0, s>>>(args);
}

template <int XT, int RT>
void launch_norm(const Args& args, bool odd, hipStream_t s) {
  if (odd) launch_rows<XT, RT, true>(args, s);
  else launch_rows<XT, RT, false>(args, s);
}

bool float_code(int dt) { return dt == CBQ_F32 || dt == CBQ_F16 || dt == CBQ_BF16; }
bool element_aligned(const void* p, int dt) { return aligned(p, dt == CBQ_F32 ? 4 : 2); }

}  // namespace
}  // namespace cbq

using namespace cbq;

extern "C" int cbq_norm(const cbq_norm_args* p, cbq_stream_t stream) {
  clear_error();
  CBQ_REQUIRE(p, "cbq_norm: args is null");
  Args args = {*p, {}, 0};
  const cbq_norm_args& a = args.a;
  CBQ_REQUIRE(a.tokens >= 0 && a.hidden >= 0, "cbq_norm: negative shape");
  CBQ_REQUIRE(a.tokens < (1LL << 31) && a.hidden < (1LL << 31), "cbq_norm: tokens and hidden must be below 2^31");
  CBQ_REQUIRE(float_code(a.x_dtype), "cbq_norm: unsupported x dtype %d", a.x_dtype);
  CBQ_REQUIRE(!a.residual || a.residual_dtype == a.x_dtype || a.residual_dtype == CBQ_F32,
              "cbq_norm: the residual must have x's dtype or float32, got %d", a.residual_dtype);
  CBQ_REQUIRE(!a.out || a.out_dtype == CBQ_I8 || float_code(a.out_dtype), "cbq_norm: unsupported out dtype %d",
              a.out_dtype);
  const bool params = a.weight || a.bias || a.post_weight || a.post_bias;
  CBQ_REQUIRE(!params || float_code(a.param_dtype), "cbq_norm: unsupported parameter dtype %d", a.param_dtype);
  CBQ_REQUIRE(!a.gate || float_code(a.gate_dtype), "cbq_norm: unsupported gate dtype %d", a.gate_dtype);
  CBQ_REQUIRE(a.kind == CBQ_NORM_RMS || a.kind == CBQ_NORM_LAYER, "cbq_norm: unknown kind %d", a.kind);
  CBQ_REQUIRE(a.residual || (!a.post && !a.gate && !a.post_weight && !a.post_bias),
              "cbq_norm: a gate and a norm after the block need a residual");
  CBQ_REQUIRE(a.post || (!a.post_weight && !a.post_bias), "cbq_norm: post_weight and post_bias need post");
  CBQ_REQUIRE(!a.gate || a.gate_channel_stride == 0 || a.gate_channel_stride == 1,
              "cbq_norm: gate_channel_stride must be 0 or 1");
  CBQ_REQUIRE(!a.gate || a.gate_token_stride >= 0, "cbq_norm: negative gate_token_stride");
  if (a.tokens == 0 || a.hidden == 0) return CBQ_OK;
  CBQ_REQUIRE(a.x && (!a.residual || a.h) && (a.residual || a.out), "cbq_norm: null pointer");
  CBQ_REQUIRE(!a.out || a.out_dtype != CBQ_I8 || a.scale, "cbq_norm: codes need scale");
  CBQ_REQUIRE(a.x_stride >= a.hidden && (!a.residual || a.residual_stride >= a.hidden),
              "cbq_norm: rows closer than hidden elements");
  CBQ_REQUIRE(element_aligned(a.x, a.x_dtype) && element_aligned(a.residual, a.residual_dtype) &&
                  element_aligned(a.h, a.residual_dtype) && element_aligned(a.weight, a.param_dtype) &&
                  element_aligned(a.bias, a.param_dtype) && element_aligned(a.post_weight, a.param_dtype) &&
                  element_aligned(a.post_bias, a.param_dtype) && element_aligned(a.gate, a.gate_dtype) &&
                  (a.out_dtype == CBQ_I8 || element_aligned(a.out, a.out_dtype)),
              "cbq_norm: tensors must be aligned to their elements");
  args.n = Norm{a.kind == CBQ_NORM_LAYER, a.eps, 1.0f / static_cast<float>(a.hidden)};
  // Inputs that the Infinity Cache cannot still hold are read past it (8192 x 8192 with a
  // residual, 268 MB: 78 us against 85), others through it (16384 x 1408, 46 MB: 19
  // against 24).
  const int x_size = a.x_dtype == CBQ_F32 ? 4 : 2, r_size = a.residual_dtype == CBQ_F32 ? 4 : 2;
  args.stream = a.tokens * a.hidden * (x_size + (a.residual ? r_size : 0)) >= 192 * 1000 * 1000;
  // Even rows: see index_of.
  auto even = [&](const void* t, int64_t stride, int size) { return aligned(t, 4) && stride * size % 4 == 0; };
  const int p_size = a.param_dtype == CBQ_F32 ? 4 : 2, g_size = a.gate_dtype == CBQ_F32 ? 4 : 2;
  bool odd = a.hidden % 8 || !even(a.x, a.x_stride, x_size) || !even(a.out, 0, 1);
  if (a.residual) odd = odd || !even(a.residual, a.residual_stride, r_size) || !even(a.h, 0, 1);
  for (const void* t : {a.weight, a.bias, a.post_weight, a.post_bias}) odd = odd || !even(t, 0, p_size);
  if (a.gate && a.gate_channel_stride) odd = odd || !even(a.gate, a.gate_token_stride, g_size);
  hipStream_t s = as_stream(stream);
  const int rt = a.residual ? a.residual_dtype : a.x_dtype;
  // A grid has fewer than 2^32 threads, up to 1024 for a row.
  constexpr int64_t kRows = 1 << 21;
  auto bytes = [](int dt) { return dt == CBQ_F32 ? 4 : dt == CBQ_I8 ? 1 : 2; };
  const int64_t H = a.hidden, tokens = a.tokens;
  for (int64_t t = 0; t < tokens; t += kRows) {
    Args part = args;
    cbq_norm_args& b = part.a;
    auto skip = [&](auto& q, int64_t elements, int dt) {
      using T = std::remove_reference_t<decltype(q)>;
      if (q) q = reinterpret_cast<T>(reinterpret_cast<uintptr_t>(q) + elements * bytes(dt));
    };
    b.tokens = std::min(kRows, tokens - t);
    skip(b.x, t * a.x_stride, a.x_dtype);
    skip(b.residual, t * a.residual_stride, rt);
    skip(b.gate, t * a.gate_token_stride, a.gate_dtype);
    skip(b.h, t * H, rt);
    skip(b.out, t * H, a.out_dtype);
    if (b.scale) b.scale += t;
    if (a.x_dtype == CBQ_F32) launch_norm<kF32, kF32>(part, odd, s);
    else if (a.x_dtype == CBQ_F16 && rt == CBQ_F16) launch_norm<kF16, kF16>(part, odd, s);
    else if (a.x_dtype == CBQ_F16) launch_norm<kF16, kF32>(part, odd, s);
    else if (rt == CBQ_BF16) launch_norm<kBF16, kBF16>(part, odd, s);
    else launch_norm<kBF16, kF32>(part, odd, s);
  }
  return launch_status("cbq_norm");
}
