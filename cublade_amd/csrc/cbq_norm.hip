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
// and written once, in chunks of 8 elements per thread (16-byte accesses, which need
// no alignment; a row's last chunk element by element). What bounds the kernel is
// memory for many tokens, and the chain of load, reductions and store for few.
// The sum of squares and the largest |v weight| are reduced together: rounding is
// monotonic, so max |v weight| rstd is the largest of the rounded products.
//
// A NaN or an infinity in a row makes its maximum NaN (maxima are taken over the bit
// patterns of absolute values, where a NaN is above everything) and with it the scale:
// the token's outputs of a product are NaN rather than those of zero codes.
#include "cbq_device.h"
#include "cbq_host.h"
#include "cublade_w8a8.h"

namespace cbq {
namespace {

typedef u32x4 __attribute__((aligned(2))) u32x4_a2;
typedef u32x2 __attribute__((aligned(1))) u32x2_a1;
typedef u32x4 __attribute__((aligned(1))) u32x4_a1;

// Eight elements of any type; of 16-bit types in a.
struct Raw { u32x4 a, b; };

template <bool NT>
__device__ __forceinline__ u32x4 ld16u(const void* p) {
  const u32x4_a2* q = static_cast<const u32x4_a2*>(p);
  return NT ? __builtin_nontemporal_load(q) : *q;
}

// Elements e .. e + 7 of a row of H; zeros from H on.
template <int DT, bool NT = false>
__device__ __forceinline__ Raw ld_raw(const void* row, int64_t e, int64_t H) {
  Raw r = {u32x4{0u, 0u, 0u, 0u}, u32x4{0u, 0u, 0u, 0u}};
  if (e + 8 <= H) {
    const char* p = static_cast<const char*>(row) + e * elem_bytes<DT>();
    r.a = ld16u<NT>(p);
    if constexpr (DT == kF32) r.b = ld16u<NT>(p + 16);
  } else if (e < H) {
    uint32_t w[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (e + k < H) {
        if constexpr (DT == kF32) w[k] = static_cast<const uint32_t*>(row)[e + k];
        else w[k >> 1] |= static_cast<uint32_t>(static_cast<const uint16_t*>(row)[e + k]) << (16 * (k & 1));
      }
    r.a = u32x4{w[0], w[1], w[2], w[3]};
    if constexpr (DT == kF32) r.b = u32x4{w[4], w[5], w[6], w[7]};
  }
  return r;
}

template <int DT>
__device__ __forceinline__ void widen(const Raw& r, float (&f)[8]) {
  Raw8<DT> t;
  t.a = make_uint4(r.a.x, r.a.y, r.a.z, r.a.w);
  if constexpr (DT == kF32) t.b = make_uint4(r.b.x, r.b.y, r.b.z, r.b.w);
  cvt8<DT>(t, f);
}

// The same for a type known at run time only (the same for all threads).
__device__ __forceinline__ Raw ld_raw(const void* row, int dt, int64_t e, int64_t H) {
  return dt == kF32 ? ld_raw<kF32>(row, e, H) : ld_raw<kF16>(row, e, H);
}
__device__ __forceinline__ void widen(const Raw& r, int dt, float (&f)[8]) {
  if (dt == kF32) widen<kF32>(r, f);
  else if (dt == kF16) widen<kF16>(r, f);
  else widen<kBF16>(r, f);
}

template <int DT>
__device__ __forceinline__ void narrow(const float (&f)[8], Raw& r) {
  if constexpr (DT == kF32) {
    r.a = u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    r.b = u32x4{__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])};
  } else {
    r.a = u32x4{pack2_out<DT>(f[0], f[1]), pack2_out<DT>(f[2], f[3]), pack2_out<DT>(f[4], f[5]),
                pack2_out<DT>(f[6], f[7])};
  }
}

template <int DT>
__device__ __forceinline__ void st_raw(void* row, int64_t e, int64_t H, const Raw& r) {
  if (e + 8 <= H) {
    char* p = static_cast<char*>(row) + e * elem_bytes<DT>();
    *reinterpret_cast<u32x4_a2*>(p) = r.a;
    if constexpr (DT == kF32) *reinterpret_cast<u32x4_a2*>(p + 16) = r.b;
  } else {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (e + k < H) {
        if constexpr (DT == kF32) static_cast<uint32_t*>(row)[e + k] = w[k];
        else static_cast<uint16_t*>(row)[e + k] = static_cast<uint16_t>(w[k >> 1] >> (16 * (k & 1)));
      }
  }
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Sum and maximum over a row's threads; every thread gets both.
struct Stat { float sum; uint32_t top; };

__device__ __forceinline__ Stat wave_stat(Stat s) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    s.sum += __shfl_xor(s.sum, o, kWave);
    const uint32_t t = __shfl_xor(s.top, o, kWave);
    s.top = s.top > t ? s.top : t;
  }
  return s;
}

// slots: one per wave, another set for each reduction of the kernel.
template <bool WAVE>
__device__ __forceinline__ Stat row_stat(Stat s, Stat* slots) {
  s = wave_stat(s);
  if constexpr (!WAVE) {
    const int waves = blockDim.x / kWave;
    if (threadIdx.x % kWave == 0) slots[threadIdx.x / kWave] = s;
    __syncthreads();
    s = slots[0];
    for (int w = 1; w < waves; ++w) {
      const Stat o = slots[w];
      s.sum += o.sum;
      s.top = s.top > o.top ? s.top : o.top;
    }
  }
  return s;
}

struct Norm {
  int layer;               // else rms
  float eps;
  int64_t H;
  float inv_h;
};

__device__ __forceinline__ float rstd_of(float ss, const Norm& n) {
  return __builtin_amdgcn_rsqf(ss * n.inv_h + n.eps);
}

// The codes of 8 values, and the row's stored scale.
__device__ __forceinline__ float row_inv(float amax) {
  return amax == amax ? inv_scale(amax, 1e-12f, kQmaxInt8) : amax;
}

struct Args {
  cbq_norm_args a;
  Norm n;
};

__device__ __forceinline__ void st_out(const cbq_norm_args& a, int64_t token, int64_t e,
                                       const float (&f)[8], float inv) {
  const int64_t H = a.hidden;
  if (a.out_dtype == CBQ_I8) {
    uint8_t* row = static_cast<uint8_t*>(a.out) + token * H;
    const uint2 q = pack8_int8(f, inv);
    if (e + 8 <= H) {
      *reinterpret_cast<u32x2_a1*>(row + e) = u32x2{q.x, q.y};
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (e + k < H) row[e + k] = static_cast<uint8_t>((k < 4 ? q.x : q.y) >> (8 * (k & 3)));
    }
    return;
  }
  Raw r;
  char* row = static_cast<char*>(a.out) + token * H * (a.out_dtype == CBQ_F32 ? 4 : 2);
  if (a.out_dtype == CBQ_F32) { narrow<kF32>(f, r); st_raw<kF32>(row, e, H, r); }
  else if (a.out_dtype == CBQ_F16) { narrow<kF16>(f, r); st_raw<kF16>(row, e, H, r); }
  else { narrow<kBF16>(f, r); st_raw<kBF16>(row, e, H, r); }
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
// waves. V chunks of 8 elements per thread.
template <int XT, int RT, int V, bool WAVE>
__global__ __launch_bounds__(WAVE ? kBlock : 1024) void k_norm(Args args) {
  const cbq_norm_args& a = args.a;
  __shared__ Stat slots[5][16];
  const int64_t H = a.hidden;
  const int64_t token = WAVE ? static_cast<int64_t>(blockIdx.x) * (kBlock / kWave) + threadIdx.x / kWave
                             : blockIdx.x;
  if (WAVE && token >= a.tokens) return;
  const int t = WAVE ? threadIdx.x % kWave : threadIdx.x;
  const int nt = WAVE ? kWave : blockDim.x;

  // All of the row's loads first.
  Raw rx[V], rr[V], rw[V];
#pragma unroll
  for (int v = 0; v < V; ++v)
    rx[v] = ld_raw<XT, true>(row_of<XT>(a.x, token, a.x_stride), (t + v * nt) * 8, H);
  if (a.residual) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      rr[v] = ld_raw<RT, true>(row_of<RT>(a.residual, token, a.residual_stride), (t + v * nt) * 8, H);
  }
  constexpr bool EARLY = V <= 2;   // longer rows have no registers to spare
  if (EARLY && a.weight) {
#pragma unroll
    for (int v = 0; v < V; ++v) rw[v] = ld_raw(a.weight, a.param_dtype, (t + v * nt) * 8, H);
  }
  float f[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v) widen<XT>(rx[v], f[v]);

  auto at = [&](int v) { return static_cast<int64_t>(t + v * nt) * 8; };
  // Elements past the row are zero.
  auto clip = [&](int v) {
    if (at(v) + 8 > H) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (at(v) + k >= H) f[v][k] = 0.0f;
    }
  };
  // layer: the mean leaves f.
  auto centre = [&](Stat* s) {
    if (!args.n.layer) return;
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += f[v][k];
    const float mean = row_stat<WAVE>({sum, 0u}, s).sum * args.n.inv_h;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[v][k] -= mean;
      clip(v);
    }
  };
  auto squares = [&] {
    float ss = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < 8; ++k) ss += f[v][k] * f[v][k];
    return ss;
  };
  // f = f p, or f + p, with a parameter of the channels.
  auto scale_by = [&](const void* p, const Raw* early) {
    if (!p) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float w[8];
      widen(early ? early[v] : ld_raw(p, a.param_dtype, at(v), H), a.param_dtype, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[v][k] *= w[k];
    }
  };
  auto shift_by = [&](const void* p) {
    if (!p) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float w[8];
      widen(ld_raw(p, a.param_dtype, at(v), H), a.param_dtype, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[v][k] += w[k];
    }
  };

  if (a.residual) {
    if (a.post) {
      centre(slots[0]);
      const float rstd = rstd_of(row_stat<WAVE>({squares(), 0u}, slots[1]).sum, args.n);
      scale_by(a.post_weight, nullptr);
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < 8; ++k) f[v][k] *= rstd;
      shift_by(a.post_bias);
    }
    if (a.gate) {
      const char* g = gate_row(a, token);
      if (a.gate_channel_stride == 0) {
        const float gv = a.gate_dtype == CBQ_F32 ? ld1<kF32>(g, 0)
                         : a.gate_dtype == CBQ_F16 ? ld1<kF16>(g, 0) : ld1<kBF16>(g, 0);
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int k = 0; k < 8; ++k) f[v][k] *= gv;
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float w[8];
          widen(ld_raw(g, a.gate_dtype, at(v), H), a.gate_dtype, w);
#pragma unroll
          for (int k = 0; k < 8; ++k) f[v][k] *= w[k];
        }
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float r[8];
      widen<RT>(rr[v], r);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[v][k] = r[k] + a.alpha * f[v][k];
      Raw o;
      narrow<RT>(f[v], o);
      st_raw<RT>(static_cast<char*>(a.h) + token * H * elem_bytes<RT>(), at(v), H, o);
      widen<RT>(o, f[v]);
      clip(v);
    }
  }
  if (!a.out) return;

  centre(slots[2]);
  Stat s = {squares(), 0u};
  scale_by(a.weight, EARLY ? rw : nullptr);
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int k = 0; k < 8; ++k) s.top = s.top > abs_bits(f[v][k]) ? s.top : abs_bits(f[v][k]);
  s = row_stat<WAVE>(s, slots[3]);
  const float rstd = rstd_of(s.sum, args.n);
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int k = 0; k < 8; ++k) f[v][k] *= rstd;
  float amax = __uint_as_float(s.top) * rstd, inv = 0.0f;
  if (a.bias) {
    shift_by(a.bias);
    if (a.out_dtype == CBQ_I8) {
      uint32_t top = 0u;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        clip(v);
#pragma unroll
        for (int k = 0; k < 8; ++k) top = top > abs_bits(f[v][k]) ? top : abs_bits(f[v][k]);
      }
      amax = __uint_as_float(row_stat<WAVE>({0.0f, top}, slots[4]).top);
    }
  }
  if (a.out_dtype == CBQ_I8) {
    inv = row_inv(amax);
    if (t == 0) a.scale[token] = 1.0f / inv;
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (at(v) < H) st_out(a, token, at(v), f[v], inv);
}

// Rows too long for registers: a workgroup of 1024 per row, which reads its row again
// for each sum (h from where this thread stored it).
template <int XT, int RT>
__global__ __launch_bounds__(1024) void k_norm_long(Args args) {
  const cbq_norm_args& a = args.a;
  __shared__ Stat slots[6][16];
  const int64_t H = a.hidden, token = blockIdx.x;
  const char* x = row_of<XT>(a.x, token, a.x_stride);
  char* h = static_cast<char*>(a.h) + (a.residual ? token * H * elem_bytes<RT>() : 0);
  const char* g = a.gate ? gate_row(a, token) : nullptr;
  auto each = [&](auto&& fn) {
    for (int64_t e = threadIdx.x * 8; e < H; e += 1024 * 8) fn(e, static_cast<int>(H - e < 8 ? H - e : 8));
  };
  auto ld_p = [&](const void* p, int dt, int64_t e, float (&w)[8]) { widen(ld_raw(p, dt, e, H), dt, w); };
  auto ld_x = [&](int64_t e, float (&f)[8]) { widen<XT>(ld_raw<XT>(x, e, H), f); };
  auto ld_v = [&](int64_t e, float (&f)[8]) {   // what the last norm is of
    if (a.residual) widen<RT>(ld_raw<RT>(h, e, H), f);
    else ld_x(e, f);
  };
  auto moments = [&](auto&& ld, Stat* s0, Stat* s1, float& mean) {
    mean = 0.0f;
    float f[8];
    if (args.n.layer) {
      float sum = 0.0f;
      each([&](int64_t e, int) {
        ld(e, f);
        for (int k = 0; k < 8; ++k) sum += f[k];
      });
      mean = row_stat<false>({sum, 0u}, s0).sum * args.n.inv_h;
    }
    float ss = 0.0f;
    each([&](int64_t e, int n) {
      ld(e, f);
      for (int k = 0; k < 8; ++k)
        if (k < n) ss += (f[k] - mean) * (f[k] - mean);
    });
    return rstd_of(row_stat<false>({ss, 0u}, s1).sum, args.n);
  };
  auto normed = [&](float (&f)[8], int64_t e, float mean, float rstd, const void* w, const void* b) {
    float p[8];
    for (int k = 0; k < 8; ++k) f[k] -= mean;
    if (w) {
      ld_p(w, a.param_dtype, e, p);
      for (int k = 0; k < 8; ++k) f[k] *= p[k];
    }
    for (int k = 0; k < 8; ++k) f[k] *= rstd;
    if (b) {
      ld_p(b, a.param_dtype, e, p);
      for (int k = 0; k < 8; ++k) f[k] += p[k];
    }
  };
  float mean, rstd;
  if (a.residual) {
    if (a.post) rstd = moments(ld_x, slots[0], slots[1], mean);
    each([&](int64_t e, int) {
      float f[8], r[8], w[8];
      ld_x(e, f);
      if (a.post) normed(f, e, mean, rstd, a.post_weight, a.post_bias);
      if (g && a.gate_channel_stride) ld_p(g, a.gate_dtype, e, w);
      else if (g) {
        ld_p(g, a.gate_dtype, 0, w);
        for (int k = 1; k < 8; ++k) w[k] = w[0];
      }
      widen<RT>(ld_raw<RT>(row_of<RT>(a.residual, token, a.residual_stride), e, H), r);
      for (int k = 0; k < 8; ++k) f[k] = r[k] + a.alpha * (g ? f[k] * w[k] : f[k]);
      Raw o;
      narrow<RT>(f, o);
      st_raw<RT>(h, e, H, o);
    });
  }
  if (!a.out) return;
  rstd = moments(ld_v, slots[2], slots[3], mean);
  float inv = 0.0f;
  if (a.out_dtype == CBQ_I8) {
    uint32_t top = 0u;
    each([&](int64_t e, int n) {
      float f[8];
      ld_v(e, f);
      normed(f, e, mean, rstd, a.weight, a.bias);
      for (int k = 0; k < 8; ++k)
        if (k < n && abs_bits(f[k]) > top) top = abs_bits(f[k]);
    });
    inv = row_inv(__uint_as_float(row_stat<false>({0.0f, top}, slots[4]).top));
    if (threadIdx.x == 0) a.scale[token] = 1.0f / inv;
  }
  each([&](int64_t e, int) {
    float f[8];
    ld_v(e, f);
    normed(f, e, mean, rstd, a.weight, a.bias);
    st_out(a, token, e, f, inv);
  });
}

template <int XT, int RT>
void launch_norm(const Args& args, hipStream_t s) {
  const int64_t chunks = cdiv(args.a.hidden, 8), tokens = args.a.tokens;
  const unsigned rows = static_cast<unsigned>(tokens);
  const unsigned quads = static_cast<unsigned>(cdiv(tokens, kBlock / kWave));
  auto threads = [](int64_t per) { return static_cast<unsigned>(cdiv(per, kWave) * kWave); };
  // One chunk per thread for few tokens, where the chain of a row counts; two for
  // many, where more rows in flight and fewer reductions do.
  const bool many = tokens > 2 * device_cus();
  if (chunks <= kWave) k_norm<XT, RT, 1, true><<<quads, kBlock, 0, s>>>(args);
  else if (chunks <= 2 * kWave) k_norm<XT, RT, 2, true><<<quads, kBlock, 0, s>>>(args);
  else if (chunks <= 1024 && !(many && chunks > 256)) k_norm<XT, RT, 1, false><<<rows, threads(chunks), 0, s>>>(args);
  else if (chunks <= 2048) k_norm<XT, RT, 2, false><<<rows, threads(cdiv(chunks, 2)), 0, s>>>(args);
  else if (chunks <= 4096) k_norm<XT, RT, 4, false><<<rows, threads(cdiv(chunks, 4)), 0, s>>>(args);
  else k_norm_long<XT, RT><<<rows, 1024, 0, s>>>(args);
}

bool float_code(int dt) { return dt == CBQ_F32 || dt == CBQ_F16 || dt == CBQ_BF16; }
bool element_aligned(const void* p, int dt) { return aligned(p, dt == CBQ_F32 ? 4 : 2); }

}  // namespace
}  // namespace cbq

using namespace cbq;

extern "C" int cbq_norm(const cbq_norm_args* p, cbq_stream_t stream) {
  clear_error();
  CBQ_REQUIRE(p, "cbq_norm: args is null");
  Args args = {*p, {}};
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
  args.n = Norm{a.kind == CBQ_NORM_LAYER, a.eps, a.hidden, 1.0f / static_cast<float>(a.hidden)};
  hipStream_t s = as_stream(stream);
  const int rt = a.residual ? a.residual_dtype : a.x_dtype;
  if (a.x_dtype == CBQ_F32) launch_norm<kF32, kF32>(args, s);
  else if (a.x_dtype == CBQ_F16 && rt == CBQ_F16) launch_norm<kF16, kF16>(args, s);
  else if (a.x_dtype == CBQ_F16) launch_norm<kF16, kF32>(args, s);
  else if (rt == CBQ_BF16) launch_norm<kBF16, kBF16>(args, s);
  else launch_norm<kBF16, kF32>(args, s);
  return launch_status("cbq_norm");
}
