// cbq_kv_attend.hip - attention over the 8-bit paged key/value cache.
//
// For a query row q and its visible keys j, with scale c, K codes k_j of scale
// ks(j) and V codes v_j of scale vs(j) (one scale per page and kv head):
//   y_j = (c log2 e) ks(j) (q . k_j) + log2 vs(j)
//   m   = max_j y_j,  w_j = 2^(y_j - m)            (in [0, 1], rounded to fp16)
//   o   = sum_j w_j v_j / sum_j w_j / vs(j)
// The value scale sits in the exponent, so the weights of the product with the
// codes stay in [0, 1] whatever the scales are, and neither codes nor
// accumulators are ever multiplied by a scale. Codes are exact in fp16 (INT8
// up to 127, E4M3 entirely), so both products run on the fp16 matrix cores
// with fp32 sums and only the queries (bf16 ones are scaled to fp16 by a power
// of two per row) and the weights are rounded.
//
// The matrix products compute S^T = K q^T and O^T = V^T w^T. In S^T's result
// layout a lane holds 4 consecutive rows (keys) of one column (query row) per
// tile; which cached token stands in which row is free, and chosen so that the
// lane's keys are 16 consecutive tokens: what it has is then the second
// product's operand as it is, and its V^T operand is 16 consecutive bytes of
// one dimension in the transposed page. No operand passes through LDS.
#include <algorithm>
#include <type_traits>

#include "cbq_kv.h"
#include "cbq_mfma.h"

namespace cbq {
namespace {

constexpr float kNegInf = -__builtin_inff();
constexpr float kLn2 = 0.69314718055994531f;
constexpr float kLog2e = 1.44269504088896341f;
constexpr int kMaxSplits = 64;      // one lane of the joining wave each
constexpr int kRowTile = 16;        // query rows of a workgroup
constexpr int kStep = 64;           // keys of a wave's step
// The running maximum is raised only when a tile exceeds it by 2^8: weights
// then stay below 2^8, far from fp16's 65504, and most steps do not touch the
// accumulators.
constexpr float kRaise = 8.0f;
// A scale below this counts as this: log2 of a page scale of 0 (a page of a
// zero-filled pool, which stands for zeros) must stay finite. append's scales
// are at least 1e-12 / 448 > 2^-49.
constexpr float kTinyScale = 0x1p-64f;

struct KvAttendArg {
  KvBatch m;
  const char* q;
  int64_t qts, qhs;        // bytes
  const uint8_t* kc;
  const uint8_t* vc;
  const float* ks;
  const float* vs;
  char* out;
  float* lse;
  float* po;               // [splits, tokens * hq, d] unnormalised partial outputs
  float2* pml;             // [splits, tokens * hq] their (m, sum)
  int64_t window;
  float scale_log2e;
  int hkv, hq, rep, d, page;
  int causal, bf16, splits, tiles;
};

// 8 codes -> 8 exact fp16.
template <int ST>
__device__ __forceinline__ u32x4 widen8(uint32_t a, uint32_t b) {
  if constexpr (ST == kKvInt8) {
    // code ^ 0x80 = code + 128 as a byte; under the high byte 0x64 it is the
    // fp16 number 1024 + 128 + code
    const f16x2 off = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    const uint32_t ua = a ^ 0x80808080u, ub = b ^ 0x80808080u;
    auto two = [&](uint32_t u, uint32_t sel) {
      const uint32_t w = __builtin_amdgcn_perm(0x64646464u, u, sel);
      return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, w) - off);
    };
    return u32x4{two(ua, 0x04010400u), two(ua, 0x04030402u), two(ub, 0x04010400u),
                 two(ub, 0x04030402u)};
  } else {
    auto two = [](uint32_t u, auto hi) {
      return __builtin_bit_cast(uint32_t,
                                __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, 1.0f, hi.value));
    };
    return u32x4{two(a, std::false_type{}), two(a, std::true_type{}), two(b, std::false_type{}),
                 two(b, std::true_type{})};
  }
}

// Over the 4 lane groups of 16 that hold one query row's keys.
__device__ __forceinline__ float max_groups(float v) {
  const uint32_t u = __float_as_uint(v);
  const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(u, u, false, false));
  v = fmaxf(__uint_as_float(a.x), __uint_as_float(a.y));
  const uint32_t w = __float_as_uint(v);
  const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(w, w, false, false));
  return fmaxf(__uint_as_float(b.x), __uint_as_float(b.y));
}

__device__ __forceinline__ float sum_groups(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// Bytes of a word that are E4M3 NaN (0x7f, 0xff), as a mask of their high bits.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// The keys a query row sees: [lo, hi).
struct KeyRange {
  int64_t lo, hi;
};

__device__ __forceinline__ KeyRange keys_of(const KvAttendArg& a, int64_t len, int64_t n,
                                            int64_t i) {
  KeyRange r;
  r.lo = 0;
  r.hi = len;
  if (a.causal) {
    const int64_t end = len - n + i + 1;
    r.hi = end < 0 ? 0 : end;
    if (a.window > 0 && end > a.window) r.lo = end - a.window;
  }
  return r;
}

// Writes one row's 4 outputs (finished or partial).
__device__ __forceinline__ void put_row(const KvAttendArg& a, int64_t row, int split, int d0,
                                        f4 o, float m, float l, bool bad) {
  if (a.splits > 1) {
    *reinterpret_cast<f4*>(a.po + (static_cast<int64_t>(split) * a.m.tokens * a.hq + row) * a.d + d0) = o;
    if (d0 == 0)
      a.pml[static_cast<int64_t>(split) * a.m.tokens * a.hq + row] =
          bad ? make_float2(0.0f, __builtin_nanf("")) : make_float2(m, l);
    return;
  }
  const bool none = m == kNegInf;
  float inv = none ? 0.0f : 1.0f / l;
  if (bad) inv = __builtin_nanf("");
  const float f[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  uint2 w;
  if (a.bf16) w = make_uint2(pack2_out<kBF16>(f[0], f[1]), pack2_out<kBF16>(f[2], f[3]));
  else w = make_uint2(pack2_out<kF16>(f[0], f[1]), pack2_out<kF16>(f[2], f[3]));
  *reinterpret_cast<uint2*>(a.out + (row * a.d + d0) * 2) = w;
  if (d0 == 0 && a.lse != nullptr)
    a.lse[row] = bad ? __builtin_nanf("") : none ? kNegInf : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

struct RowTiles {
  int rep;
  __device__ int64_t operator()(const KvSeq& s) const {
    return (s.n * rep + kRowTile - 1) / kRowTile;
  }
};

// One workgroup: 16 query rows of one kv head (row = new token * rep + head in
// the group) and one range of the keys. Its 4 waves take steps of 64 keys in
// turn, each with its own maximum, sum and accumulators, joined at the end.
// DP: head_dim padded to a multiple of 64; EXACT: head_dim is DP.
template <int ST, int DP, bool EXACT>
__global__ __launch_bounds__(kBlock, DP <= 128 ? 2 : 1) void k_kv_attend_rows(const KvAttendArg a) {
  constexpr int NC = DP / 64;      // 16-byte chunks of a key per lane
  constexpr int ND = DP / 16;      // tiles of 16 dimensions
  const int d = EXACT ? DP : a.d;
  __shared__ __attribute__((aligned(16))) float so[4][kRowTile][DP + 4];
  __shared__ float sml[4][kRowTile][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n16 = lane & 15, g = lane >> 4;

  const int split = blockIdx.x % a.splits;
  const int64_t rest = blockIdx.x / a.splits;
  const int h = rest % a.hkv;
  const int64_t item = rest / a.hkv;
  int64_t tile;
  int b;
  if (a.m.cu == nullptr) {
    b = static_cast<int>(item / a.tiles);
    tile = item % a.tiles;
  } else {
    b = kv_find(a.m, item, tile, RowTiles{a.rep});
    if (b < 0) return;
  }
  const KvSeq s = kv_seq(a.m, b);
  const int64_t cap = static_cast<int64_t>(a.m.max_pages) << a.m.page_shift;
  const bool bad = s.len > cap;      // keys that no page can hold
  const int64_t len = s.len < 0 ? 0 : bad ? cap : s.len;
  const int64_t rows = s.n * a.rep;
  const int64_t r_first = tile * kRowTile;
  const int64_t r_last = r_first + kRowTile - 1 < rows ? r_first + kRowTile - 1 : rows - 1;
  const int64_t r = r_first + n16;
  const bool has_row = r < rows;
  const int64_t ti = r / a.rep;      // the row's new token
  const int head = h * a.rep + static_cast<int>(r - ti * a.rep);
  const KeyRange mine = keys_of(a, len, s.n, ti);
  const KeyRange kf = keys_of(a, len, s.n, r_first / a.rep);
  const KeyRange kl = keys_of(a, len, s.n, r_last / a.rep);

  const int64_t kb = kf.lo / kStep, ke = (kl.hi + kStep - 1) / kStep;
  int64_t per = (ke - kb + a.splits - 1) / a.splits;
  per = per < 4 ? 4 : per;
  const int64_t s0 = kb + split * per;
  const int64_t s1 = s0 + per < ke ? s0 + per : ke;

  f4 o[ND] = {};
  float m = kNegInf, l = 0.0f;

  if (s0 + wave < s1) {
    // the queries as fp16, and what the scores are multiplied by
    u32x4 qf[2 * NC];
    float cq = a.scale_log2e;
    {
      float f[2 * NC][8];
      float amax = 0.0f;
      const char* qp = a.q + (s.tok0 + ti) * a.qts + head * a.qhs;
#pragma unroll
      for (int c = 0; c < 2 * NC; ++c) {
        const int d0 = 64 * (c >> 1) + 16 * g + 8 * (c & 1);
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (has_row && d0 < d) raw = *reinterpret_cast<const uint4*>(qp + 2 * d0);
        if (a.bf16) {
          Raw8<kBF16> w{raw};
          cvt8<kBF16>(w, f[c]);
          amax = absmax8(f[c], amax);
        } else {
          qf[c] = u32x4{raw.x, raw.y, raw.z, raw.w};
        }
      }
      if (a.bf16) {
        amax = max_groups(amax);
        const int e = static_cast<int>(__float_as_uint(amax) >> 23);   // biased exponent
        float up = 1.0f;
        if (e > 0 && e < 254) {     // amax * up in [1, 2)
          up = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
          cq *= __uint_as_float(static_cast<uint32_t>(e) << 23);
        }
#pragma unroll
        for (int c = 0; c < 2 * NC; ++c) {
          float x[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = f[c][k] * up;
          const uint4 w = pack8_out<kF16>(x);
          qf[c] = u32x4{w.x, w.y, w.z, w.w};
        }
      }
    }

    const int64_t last_block = (kl.hi - 1) >> 4;
    auto block_of = [&](int64_t st, int quarter) {
      const int64_t bl = st * 4 + quarter;
      return bl < last_block ? bl : last_block;
    };
    auto page_of = [&](int64_t bl) { return a.m.table[b * a.m.tstride + ((bl << 4) >> a.m.page_shift)]; };
    auto valid = [&](int id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(a.m.num_pages); };
    u32x4 kr[4][NC];
    float ksc = 0.0f, vsc = 1.0f;
    int id_v = 0;
    // Row r of tile t is the key 16 (r / 4) + 4 t + r % 4 of the step.
    auto load_k = [&](int64_t st, int idk, int idv) {
      const int64_t bl = block_of(st, n16 >> 2);
      const int64_t at = static_cast<int64_t>(valid(idk) ? idk : 0) * a.hkv + h;
      const uint8_t* p = a.kc + (at * a.page + ((bl << 4) & (a.page - 1)) + (n16 & 3)) * d + 16 * g;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          kr[t][c] = u32x4{0, 0, 0, 0};
          if (64 * c + 16 * g < d) kr[t][c] = *reinterpret_cast<const u32x4*>(p + 4 * t * d + 64 * c);
        }
      const int64_t sat = static_cast<int64_t>(valid(idv) ? idv : 0) * a.hkv + h;
      ksc = valid(idv) ? a.ks[sat] : __builtin_nanf("");
      vsc = a.vs[sat];
      id_v = valid(idv) ? idv : 0;
    };
    load_k(s0 + wave, page_of(block_of(s0 + wave, n16 >> 2)), page_of(block_of(s0 + wave, g)));
    int next_k = 0, next_v = 0;
    if (s0 + wave + 4 < s1) {
      next_k = page_of(block_of(s0 + wave + 4, n16 >> 2));
      next_v = page_of(block_of(s0 + wave + 4, g));
    }

    for (int64_t st = s0 + wave; st < s1; st += 4) {
      const int64_t tb = st * kStep;
      // this step's values
      u32x4 vr[ND];
      {
        const int64_t bl = block_of(st, g);
        const uint8_t* p = a.vc + ((static_cast<int64_t>(id_v) * a.hkv + h) * d + n16) * a.page +
                           ((bl << 4) & (a.page - 1));
#pragma unroll
        for (int t = 0; t < ND; ++t) {
          vr[t] = u32x4{0, 0, 0, 0};
          if (16 * t < d) vr[t] = *reinterpret_cast<const u32x4*>(p + 16 * t * a.page);
        }
      }
      // scores of 64 keys: lane (n16, g) gets keys tb + 16 g + 4 t + i of row n16
      f4 sc[4] = {};
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          sc[t] = mfma16x16x32<kF16>(widen8<ST>(kr[t][c].x, kr[t][c].y), qf[2 * c], sc[t]);
          sc[t] = mfma16x16x32<kF16>(widen8<ST>(kr[t][c].z, kr[t][c].w), qf[2 * c + 1], sc[t]);
        }
      const float cks = cq * ksc;
      const float vsx = vsc < kTinyScale ? kTinyScale : vsc;
      if (st + 4 < s1) {
        load_k(st + 4, next_k, next_v);
        if (st + 8 < s1) {
          next_k = page_of(block_of(st + 8, n16 >> 2));
          next_v = page_of(block_of(st + 8, g));
        }
      }
      const float lvs = __builtin_amdgcn_logf(vsx);
      float y[4][4];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[t][i] = __builtin_fmaf(sc[t][i], cks, lvs);
      const bool masked = tb + kStep > kf.hi || tb < kl.lo;   // the same in the whole workgroup
      if (masked) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int64_t j = tb + 16 * g + 4 * t + i;
            if (j < mine.lo || j >= mine.hi) y[t][i] = kNegInf;
          }
      }
      float mx = y[0][0];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, y[t][i]);
      mx = max_groups(mx);
      const bool raise = mx > m + kRaise;
      if (__any(raise)) {
        const float to = raise ? mx : m;
        const float f = raise ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
        m = to;
        l *= f;
#pragma unroll
        for (int t = 0; t < ND; ++t) o[t] *= f;
      }
      const float ref = m == kNegInf ? 0.0f : m;
      float sum = 0.0f;
      uint32_t pw[8];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = __builtin_amdgcn_exp2f(y[t][i] - ref);
          sum += w[i];
        }
        pw[2 * t] = pack2_out<kF16>(w[0], w[1]);
        pw[2 * t + 1] = pack2_out<kF16>(w[2], w[3]);
      }
      // a lane whose keys are all masked adds nothing, whatever its scale is
      l += sum == 0.0f ? 0.0f : sum * (1.0f / vsx);
      const u32x4 p0 = {pw[0], pw[1], pw[2], pw[3]}, p1 = {pw[4], pw[5], pw[6], pw[7]};
      if constexpr (ST == kKvFp8) {
        // NaN codes must reach only the rows that see their key (0 x NaN is NaN)
        if (masked) {
          uint32_t any = 0;
#pragma unroll
          for (int t = 0; t < ND; ++t)
            any |= nan_bytes(vr[t].x) | nan_bytes(vr[t].y) | nan_bytes(vr[t].z) | nan_bytes(vr[t].w);
          if (__any(any != 0)) {
            u32x4 seen0, seen1;   // 1 where the row sees the key
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              uint32_t w = 0;
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int64_t j = tb + 16 * g + 2 * e + k;
                if (j >= mine.lo && j < mine.hi) w |= 0x3c00u << (16 * k);
              }
              if (e < 4) seen0[e] = w;
              else seen1[e - 4] = w;
            }
#pragma unroll
            for (int t = 0; t < ND; ++t) {
              u32x4 ind;          // 0x38 = 1.0 in E4M3 at NaN codes
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t nb = nan_bytes(vr[t][k]) >> 7;
                ind[k] = nb * 0x38u;
                vr[t][k] &= ~(nb * 0xffu);
              }
              f4 cnt = {};
              cnt = mfma16x16x32<kF16>(widen8<ST>(ind.x, ind.y), seen0, cnt);
              cnt = mfma16x16x32<kF16>(widen8<ST>(ind.z, ind.w), seen1, cnt);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (cnt[k] > 0.0f) o[t][k] = __builtin_nanf("");
            }
          }
        }
      }
#pragma unroll
      for (int t = 0; t < ND; ++t) {
        o[t] = mfma16x16x32<kF16>(widen8<ST>(vr[t].x, vr[t].y), p0, o[t]);
        o[t] = mfma16x16x32<kF16>(widen8<ST>(vr[t].z, vr[t].w), p1, o[t]);
      }
    }
    l = sum_groups(l);
  }

  // join the 4 waves
  if (g == 0) {
    sml[wave][n16][0] = m;
    sml[wave][n16][1] = l;
  }
#pragma unroll
  for (int t = 0; t < ND; ++t) *reinterpret_cast<f4*>(&so[wave][n16][16 * t + 4 * g]) = o[t];
  __syncthreads();
  const int row = threadIdx.x >> 4;
  const int64_t rr = r_first + row;
  if (rr >= rows) return;
  float mm = kNegInf, ll = 0.0f, f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sml[w][row][0]);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = sml[w][row][0] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(sml[w][row][0] - mm);
    ll += sml[w][row][1] * f[w];
  }
  const int64_t tok = s.tok0 + rr / a.rep;
  const int64_t orow = tok * a.hq + h * a.rep + rr % a.rep;
  for (int d0 = 4 * (threadIdx.x & 15); d0 < d; d0 += 64) {
    f4 v = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) v += *reinterpret_cast<const f4*>(&so[w][row][d0]) * f[w];
    put_row(a, orow, split, d0, v, mm, ll, bad);
  }
}

// Joins the splits' partial results: one wave per row.
__global__ __launch_bounds__(kBlock) void k_kv_attend_join(const KvAttendArg a, int64_t rows) {
  const int lane = threadIdx.x & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  float2 ml = make_float2(kNegInf, 0.0f);
  if (lane < a.splits) ml = a.pml[lane * rows + row];
  float m = ml.x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float f = ml.x == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ml.x - m);
  float l = ml.y * f;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o, 64);
  const int d0 = 4 * lane;
  f4 acc = {};
  for (int s = 0; s < a.splits; ++s) {
    const float fs = __shfl(f, s, 64);   // with all lanes active: those past d have a split's factor
    if (fs != 0.0f && d0 < a.d)
      acc += *reinterpret_cast<const f4*>(a.po + (s * rows + row) * a.d + d0) * fs;
  }
  KvAttendArg one = a;
  one.splits = 1;
  if (d0 < a.d) put_row(one, row, 0, d0, acc, m, l, false);
}

int padded_dim(int d) { return (d + 63) / 64 * 64; }

// Workgroups for whole rows, before the keys are split.
int64_t row_items(const cbq_kv_batch* b, int rep) {
  if (b->cu == nullptr) return static_cast<int64_t>(b->batch) * cdiv(rep, kRowTile);
  return std::min<int64_t>(b->tokens * rep / kRowTile + b->batch, b->tokens * cdiv(rep, kRowTile));
}

int choose_splits(const cbq_kv_cache* c, const cbq_kv_batch* b, int rep, int64_t max_length) {
  const int64_t cap = static_cast<int64_t>(b->max_pages) * c->page_size;
  const int64_t len = max_length > 0 ? std::min(max_length, cap) : cap;
  const int64_t wgs = std::max<int64_t>(1, row_items(b, rep) * c->kv_heads);
  const int64_t want = cdiv(2 * device_cus(), wgs);
  const int64_t most = cdiv(cdiv(len, kStep), 4);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, most, kMaxSplits})));
}

size_t split_bytes(const cbq_kv_cache* c, const cbq_kv_batch* b, int q_heads) {
  return static_cast<size_t>(b->tokens) * q_heads * (c->head_dim + 2) * 4;
}

}  // namespace
}  // namespace cbq

using namespace cbq;

extern "C" size_t cbq_kv_attend_ws_bytes(const cbq_kv_cache* cache, const cbq_kv_batch* batch,
                                         int32_t q_heads, int64_t max_length) {
  if (cache == nullptr || batch == nullptr || cache->kv_heads <= 0 || q_heads <= 0 ||
      q_heads % cache->kv_heads != 0 || batch->tokens <= 0)
    return CBQ_WS_CTRL_BYTES;
  const int splits = choose_splits(cache, batch, q_heads / cache->kv_heads, max_length);
  return CBQ_WS_CTRL_BYTES + (splits > 1 ? splits * split_bytes(cache, batch, q_heads) : 0);
}

extern "C" int cbq_kv_attend(const cbq_kv_cache* cache, const cbq_kv_batch* batch, int dtype,
                             const cbq_kv_heads* q, int32_t q_heads, float scale, int causal,
                             int64_t window, int64_t max_length, void* ws, size_t ws_bytes,
                             void* out, float* lse, cbq_stream_t stream) {
  clear_error();
  if (int rc = kv_check_cache(cache)) return rc;
  if (int rc = kv_check_batch(batch)) return rc;
  CBQ_REQUIRE(dtype == CBQ_F16 || dtype == CBQ_BF16, "kv attend: dtype must be fp16 or bf16, got %d",
              dtype);
  CBQ_REQUIRE(q_heads > 0 && q_heads % cache->kv_heads == 0,
              "kv attend: q_heads must be a positive multiple of kv_heads %d, got %d",
              cache->kv_heads, q_heads);
  CBQ_REQUIRE(window >= 0 && (window == 0 || causal), "kv attend: a window needs causal and must not be negative");
  if (batch->tokens == 0 || batch->batch == 0) return CBQ_OK;
  if (int rc = kv_check_heads("q", q)) return rc;
  CBQ_REQUIRE(out != nullptr && aligned(out, 16), "kv attend: out must be given, 16-byte aligned");
  CBQ_REQUIRE(ws == nullptr || aligned(ws, 256), "kv attend: workspace must be 256-byte aligned");
  const int rep = q_heads / cache->kv_heads;
  KvAttendArg a = {};
  a.m = kv_batch_of(cache, batch);
  if (cache->num_pages == 0) a.m.max_pages = 0;   // nothing to read: sequences with tokens give NaN
  a.q = static_cast<const char*>(q->data);
  a.qts = 2 * q->token_stride;
  a.qhs = 2 * q->head_stride;
  a.kc = static_cast<const uint8_t*>(cache->k);
  a.vc = static_cast<const uint8_t*>(cache->v);
  a.ks = cache->k_scale;
  a.vs = cache->v_scale;
  a.out = static_cast<char*>(out);
  a.lse = lse;
  a.window = window;
  a.scale_log2e = scale * kLog2e;
  a.hkv = cache->kv_heads;
  a.hq = q_heads;
  a.rep = rep;
  a.d = cache->head_dim;
  a.page = cache->page_size;
  a.causal = causal != 0;
  a.bf16 = dtype == CBQ_BF16;
  a.tiles = static_cast<int>(cdiv(rep, kRowTile));
  int splits = choose_splits(cache, batch, rep, max_length);
  const size_t each = split_bytes(cache, batch, q_heads);
  const size_t room = ws != nullptr && ws_bytes > CBQ_WS_CTRL_BYTES ? ws_bytes - CBQ_WS_CTRL_BYTES : 0;
  splits = static_cast<int>(std::min<size_t>(splits, room / each));
  if (splits < 1) splits = 1;
  a.splits = splits;
  const int64_t rows = batch->tokens * q_heads;
  if (splits > 1) {
    a.po = reinterpret_cast<float*>(static_cast<char*>(ws) + CBQ_WS_CTRL_BYTES);
    a.pml = reinterpret_cast<float2*>(a.po + static_cast<int64_t>(splits) * rows * a.d);
  }
  const int64_t blocks = row_items(batch, rep) * a.hkv * splits;
  CBQ_REQUIRE(blocks < (int64_t{1} << 31), "kv attend: too many tokens for one call");
  const dim3 grid(static_cast<uint32_t>(blocks));
  hipStream_t st = as_stream(stream);
  auto launch = [&](auto stc) {
    constexpr int ST = decltype(stc)::value;
    auto one = [&](auto dpc) {
      constexpr int DP = decltype(dpc)::value;
      if (a.d == DP) k_kv_attend_rows<ST, DP, true><<<grid, kBlock, 0, st>>>(a);
      else k_kv_attend_rows<ST, DP, false><<<grid, kBlock, 0, st>>>(a);
    };
    switch (padded_dim(a.d)) {
      case 64: one(std::integral_constant<int, 64>{}); break;
      case 128: one(std::integral_constant<int, 128>{}); break;
      case 192: one(std::integral_constant<int, 192>{}); break;
      default: one(std::integral_constant<int, 256>{}); break;
    }
  };
  if (cache->store == CBQ_KV_INT8) launch(std::integral_constant<int, kKvInt8>{});
  else launch(std::integral_constant<int, kKvFp8>{});
  if (int rc = launch_status("cbq_kv_attend")) return rc;
  if (splits > 1) {
    k_kv_attend_join<<<dim3(static_cast<uint32_t>(cdiv(rows, 4))), kBlock, 0, st>>>(a, rows);
    return launch_status("cbq_kv_attend");
  }
  return CBQ_OK;
}
