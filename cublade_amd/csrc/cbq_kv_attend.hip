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
// of two per row) and the weights are rounded: by 2^-11 of each, and below fp16's
// normal range by 2^-25 of the row's largest. The sum takes them before that.
//
// The matrix products compute S^T = K q^T and O^T = V^T w^T. In S^T's result
// layout a lane holds 4 consecutive rows (keys) of one column (query row) per
// tile; which cached token stands in which row is free, and chosen so that the
// lane's keys are consecutive tokens (16 in k_kv_attend_rows, 8 in
// k_kv_attend_long): what it has is then the second product's operand as it is,
// and its V^T operand is consecutive codes of one dimension in the transposed
// page. The weights never leave their registers.
//
// Measured on MI355X, one call in a stream of calls (a copy reaches 5.1 TB/s, an
// fp16 matrix product 1.15 PFLOP/s):
//   32 query heads over 8 kv heads of 128, INT8, pages of 64 tokens:
//     one token over 131077            52 us, 5.2 TB/s
//     a prompt of 8192                579 to 609 us, 0.90 to 0.95 PFLOP/s
//   128 tokens over 900 .. 1100 each, 16 heads of 64   44 us, 5.9 TB/s
//   64 tokens over 100 .. 8000 each, FP8, pages of 16  113 us, 4.2 TB/s
//   FP8, 2048 tokens of a prompt over 32768            1.11 to 1.15 ms, 0.92 to 0.96 PFLOP/s
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
// k_kv_attend_long: the most that a lane's 32 weights of a step may sum to
// before the maximum is raised (none is past fp16's range then).
constexpr float kMostWeight = 0x1p14f;
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
  float* po;               // [splits, prows, d] unnormalised partial outputs
  float2* pml;             // [splits, prows] their (m, sum)
  int64_t prows;           // partial rows: items * hkv * rows of a tile
  float scale_log2e;
  int hkv, hq, rep, d, page;
  int causal, bf16, negate, splits;
  int window;              // 0: none
  int tile_rows;           // query rows of a workgroup
  int items;               // row tiles of this launch, at most
  uint32_t tiles;          // workgroups of them; those behind: put_rest
  int row_min, row_max;       // this launch's sequences have row_min .. row_max rows
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

// v, hidden from the optimiser: what is computed from it stays where it is (the
// masks of rare steps would otherwise be prepared in every step).
__device__ __forceinline__ int opaque(int v) {
  asm("" : "+v"(v));
  return v;
}

__device__ __forceinline__ float read_lane(float v, int l) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), l));
}

__device__ __forceinline__ float max_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(u, u, false, false));
  return fmaxf(__uint_as_float(a.x), __uint_as_float(a.y));
}

// Bytes of a word that are E4M3 NaN (0x7f, 0xff), as a mask of their high bits.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// The keys a query row sees: [lo, hi). (Lengths are int32, and a call's rows of
// one kv head fewer than 2^31.)
struct KeyRange {
  int lo, hi;
};

// Tokens that a row of the page table can hold (key indices and ends of steps
// stay int32).
__device__ __forceinline__ int64_t capacity(const KvAttendArg& a) {
  const int64_t c = static_cast<int64_t>(a.m.max_pages) << a.m.page_shift;
  return c < INT32_MAX - 1024 ? c : INT32_MAX - 1024;
}

// A sequence's length as the kernels use it; bad: it has keys that no page can hold.
struct KvLen {
  int len;
  bool bad;
};

__device__ __forceinline__ KvLen len_of(const KvAttendArg& a, const KvSeq& s) {
  const int64_t cap = capacity(a);
  const bool bad = s.len > cap;
  return {static_cast<int>(s.len < 0 ? 0 : bad ? cap : s.len), bad};
}

__device__ __forceinline__ KeyRange keys_of(const KvAttendArg& a, int len, int n, int i) {
  KeyRange r;
  r.lo = 0;
  r.hi = len;
  if (a.causal) {
    const int end = len - n + i + 1;
    r.hi = end < 0 ? 0 : end;
    if (a.window > 0 && end > a.window) r.lo = end - a.window;
  }
  return r;
}

// Writes 4 outputs of one row: finished ones, or the partial row `prow` of a
// split of the keys. none: the row sees no key. (Its maximum and sum do not tell:
// scores that are all -infinity leave both as they began, and their softmax is NaN,
// as o / l = 0 / 0 is here.)
__device__ __forceinline__ void put_row(const KvAttendArg& a, int64_t row, int64_t prow, int split,
                                        int d0, f4 o, float m, float l, bool none, bool bad) {
  if (a.splits > 1) {
    const int64_t at = split * a.prows + prow;
    *reinterpret_cast<f4*>(a.po + at * a.d + d0) = o;
    if (d0 == 0) a.pml[at] = bad ? make_float2(0.0f, __builtin_nanf("")) : make_float2(m, l);
    return;
  }
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

// Outputs of the tokens that belong to no sequence, [0, cu[0]) and [cu[batch],
// tokens): zeros, log-sum-exp -infinity, as of rows that see no key. By the
// workgroups behind those of the tiles, which find nothing to do in most calls (a
// padded batch replayed from a graph has such tokens). Drafted tokens take 0.3 us
// more for it (40.7), prompts no more; a launch of its own took 2 us. (Where each
// kernel branches to it was chosen by its time: the other way is 0.4 us slower in
// k_kv_attend_rows and 2 of 78 us in a mixed batch.)
__device__ __forceinline__ void put_rest(const KvAttendArg& a) {
  int64_t lo = a.m.cu[0], hi = a.m.cu[a.m.batch];
  lo = lo < 0 ? 0 : lo > a.m.tokens ? a.m.tokens : lo;
  hi = hi < lo ? lo : hi > a.m.tokens ? a.m.tokens : hi;
  const int64_t first = static_cast<int64_t>(blockIdx.x - a.tiles) * blockDim.x + threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x - a.tiles) * blockDim.x;
  const int64_t rest = a.m.tokens - (hi - lo);
  auto each = [&](int64_t per, auto put) {     // per: elements of a token
    for (int64_t i = first; i < rest * per; i += step) put(i < lo * per ? i : i + (hi - lo) * per);
  };
  each(static_cast<int64_t>(a.hq) * a.d / 8,
       [&](int64_t i) { reinterpret_cast<uint4*>(a.out)[i] = make_uint4(0, 0, 0, 0); });
  if (a.lse != nullptr) each(a.hq, [&](int64_t i) { a.lse[i] = kNegInf; });
}

// One row's queries as fp16 operands, N pieces of 8 dimensions (piece k from
// dim(k)), and the factor cq of its scores. bf16 queries are scaled to fp16 by a
// power of two per row (row_max: the maximum over the lanes that share the row);
// the factor takes it back. A negative scale of the scores is the queries' sign
// here, so that the factor is not negative.
template <int N, typename Dim, typename Max, typename Piece>
__device__ __forceinline__ void load_q(const KvAttendArg& a, const char* qp, bool has, Dim dim,
                                       Max row_max, float& cq, Piece piece) {
  cq = a.scale_log2e;
  float amax = 0.0f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (has && dim(k) < a.d) raw = *reinterpret_cast<const uint4*>(qp + 2 * dim(k));
    piece(k) = u32x4{raw.x, raw.y, raw.z, raw.w} ^ (a.negate ? 0x80008000u : 0u);
    if (a.bf16) {
      float f[8];
      cvt8<kBF16>(Raw8<kBF16>{raw}, f);
      amax = absmax8(f, amax);
    }
  }
  if (!a.bf16) return;
  amax = row_max(amax);
  int e = static_cast<int>(__float_as_uint(amax) >> 23);   // biased exponent
  float up = 1.0f;
  if (e > 0 && e < 255) {     // amax * up in [1, 2); in [2, 4) from 2^127, whose inverse is no normal number
    e = e < 254 ? e : 253;
    up = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
    cq *= __uint_as_float(static_cast<uint32_t>(e) << 23);
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const u32x4 r = piece(k);
    float f[8];
    cvt8<kBF16>(Raw8<kBF16>{make_uint4(r.x, r.y, r.z, r.w)}, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= up;
    const uint4 w = pack8_out<kF16>(f);
    piece(k) = u32x4{w.x, w.y, w.z, w.w};
  }
}

// A sequence's query rows (row = new token * rep + head in its group) in tiles.
struct RowTiles {
  int rep, tile_rows;
  int lo, hi;
  __device__ int operator()(const KvSeq& s) const {
    const int r = static_cast<int>(s.n) * rep;
    return r >= lo && r <= hi ? (r + tile_rows - 1) / tile_rows : 0;
  }
};

// The tile of rows with number `item` of a launch: its sequence (b < 0: there is
// no such tile) and first row.
struct KvTile {
  int b;
  KvSeq s;
  int rows, r_first;
};

__device__ __forceinline__ KvTile tile_of(const KvAttendArg& a, int item) {
  KvTile t;
  int tile;
  if (a.m.cu == nullptr) {
    const int per = (a.rep + a.tile_rows - 1) / a.tile_rows;
    t.b = item / per;
    tile = item % per;
  } else {
    t.b = kv_find(a.m, item, tile, RowTiles{a.rep, a.tile_rows, a.row_min, a.row_max});
    if (t.b < 0) return t;
  }
  t.s = kv_seq(a.m, t.b);
  t.rows = static_cast<int>(t.s.n) * a.rep;
  t.r_first = tile * a.tile_rows;
  return t;
}

// ---------------------------------------------------------------------------
// Few query rows: single tokens, drafted tokens.
// ---------------------------------------------------------------------------
// One workgroup: 16 query rows of one kv head (row = new token * rep + head in
// the group) and one range of the keys. Its 4 waves take steps of 64 keys in
// turn, each with its own maximum, sum and accumulators, joined at the end; no
// operand passes through LDS. Bound by the bytes of the codes (6.3 TB/s from one
// context length to the next) and about 25 us that a call takes before and after:
// a workgroup's chain of length, page id, codes, and the joining of its waves and
// of the ranges. The loads of a step's values and of the next step's keys are in
// flight together, 16 x 16 bytes a lane at head size 128; more of them (values a
// step ahead), more workgroups per CU or wider row tiles were slower.
// Every tile's keys are cut into equally many ranges. Parts of equal length for
// sequences of mixed lengths, found by each workgroup, even out their time but cost
// more than that: a scan over the batch takes 4 us.
// DP: head_dim padded to a multiple of 64; EXACT: head_dim is DP; NT: no other
// workgroup reads the codes, and they are loaded past the caches (5.8 instead of
// 5.2 TB/s for 128 sequences of 1000 tokens; slower where several tiles of rows
// read the same codes).
template <int ST, int DP, bool EXACT, bool NT>
__global__ __launch_bounds__(kBlock, DP <= 128 ? 2 : 1) void k_kv_attend_rows(const KvAttendArg a) {
  constexpr int NC = DP / 64;      // 16-byte chunks of a key per lane
  constexpr int ND = DP / 16;      // tiles of 16 dimensions
  const int d = EXACT ? DP : a.d;
  __shared__ __attribute__((aligned(16))) float so[4][kRowTile][DP + 4];
  __shared__ float sml[4][kRowTile][2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, g = lane >> 4;

  const int split = blockIdx.x % a.splits;
  const int rest = blockIdx.x / a.splits;
  const int h = rest % a.hkv;
  const int item = rest / a.hkv;
  const KvTile tl = tile_of(a, item < a.items ? item : INT32_MAX);
  if (tl.b < 0) {
    if (item >= a.items) put_rest(a);
    return;
  }
  const int b = tl.b;
  const KvSeq s = tl.s;
  const auto [len, bad] = len_of(a, s);
  const int rows = tl.rows, r_first = tl.r_first, n = static_cast<int>(s.n);
  const int r_last = r_first + kRowTile - 1 < rows ? r_first + kRowTile - 1 : rows - 1;
  const int r = r_first + n16;
  const bool has_row = r < rows;
  const int ti = r / a.rep;      // the row's new token
  const int head = h * a.rep + r - ti * a.rep;
  const KeyRange mine = keys_of(a, len, n, ti);
  const KeyRange kf = keys_of(a, len, n, r_first / a.rep);
  const KeyRange kl = keys_of(a, len, n, r_last / a.rep);

  const int kb = kf.lo / kStep, ke = (kl.hi + kStep - 1) / kStep;
  int per = (ke - kb + a.splits - 1) / a.splits;
  per = per < 4 ? 4 : per;
  const int s0 = kb + split * per;
  const int s1 = s0 + per < ke ? s0 + per : ke;

  f4 o[ND] = {};
  float m = kNegInf, l = 0.0f;

  if (s0 + wave < s1) {
    // the queries as fp16, and what the scores are multiplied by
    u32x4 qf[2 * NC];
    float cq;
    load_q<2 * NC>(a, a.q + (s.tok0 + ti) * a.qts + head * a.qhs, has_row,
                   [&](int c) { return 64 * (c >> 1) + 16 * g + 8 * (c & 1); },
                   [](float v) { return max_groups(v); }, cq, [&](int c) -> u32x4& { return qf[c]; });

    const int last_block = (kl.hi - 1) >> 4;
    auto block_of = [&](int st, int quarter) {
      const int bl = st * 4 + quarter;
      return bl < last_block ? bl : last_block;
    };
    auto page_of = [&](int bl) { return a.m.table[b * a.m.tstride + ((bl << 4) >> a.m.page_shift)]; };
    auto valid = [&](int id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(a.m.num_pages); };
    auto load16 = [](const uint8_t* p) {
      if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
      else return *reinterpret_cast<const u32x4*>(p);
    };
    u32x4 kr[4][NC];
    float ksc = 0.0f, vsc = 1.0f;
    int id_v = 0;
    // Row r of tile t is the key 16 (r / 4) + 4 t + r % 4 of the step.
    auto load_k = [&](int st, int idk, int idv) {
      const int bl = block_of(st, n16 >> 2);
      const int64_t at = static_cast<int64_t>(valid(idk) ? idk : 0) * a.hkv + h;
      const uint8_t* p = a.kc + (at * a.page + ((bl << 4) & (a.page - 1)) + (n16 & 3)) * d + 16 * g;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          kr[t][c] = u32x4{0, 0, 0, 0};
          if (64 * c + 16 * g < d) kr[t][c] = load16(p + 4 * t * d + 64 * c);
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

    for (int st = s0 + wave; st < s1; st += 4) {
      const int tb = st * kStep;
      // this step's values
      u32x4 vr[ND];
      {
        const int bl = block_of(st, g);
        const uint8_t* p = a.vc + ((static_cast<int64_t>(id_v) * a.hkv + h) * d + n16) * a.page +
                           ((bl << 4) & (a.page - 1));
#pragma unroll
        for (int t = 0; t < ND; ++t) {
          vr[t] = u32x4{0, 0, 0, 0};
          if (16 * t < d) vr[t] = load16(p + 16 * t * a.page);
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
            const int j = tb + 16 * g + 4 * t + i;
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
                const int j = tb + 16 * g + 2 * e + k;
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
  const int rr = r_first + row;
  if (rr >= rows) return;
  float mm = kNegInf, ll = 0.0f, f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sml[w][row][0]);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = sml[w][row][0] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(sml[w][row][0] - mm);
    ll += sml[w][row][1] * f[w];
  }
  const KeyRange seen = keys_of(a, len, n, rr / a.rep);
  const int64_t tok = s.tok0 + rr / a.rep;
  const int64_t orow = tok * a.hq + h * a.rep + rr % a.rep;
  for (int d0 = 4 * (threadIdx.x & 15); d0 < d; d0 += 64) {
    f4 v = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) v += *reinterpret_cast<const f4*>(&so[w][row][d0]) * f[w];
    put_row(a, orow, static_cast<int64_t>(item * a.hkv + h) * kRowTile + row, split, d0, v, mm, ll,
            seen.hi <= seen.lo, bad);
  }
}

// ---------------------------------------------------------------------------
// Many query rows: prompts and chunks of them.
// ---------------------------------------------------------------------------
// A workgroup takes 128 or 256 rows of one kv head, a wave 32 of them; it goes
// through the keys 64 at a time. Codes are widened to fp16 once per workgroup, on
// their way from registers to LDS (K rows [64 keys][DP], V^T rows [DP][64 keys];
// every row has 16 bytes more than it needs, so an odd number of 16-byte chunks:
// equal chunks of 16 consecutive rows lie in distinct banks, and every access is a
// base register plus a constant), in two buffers. Codes are loaded two steps ahead,
// their page ids three; one barrier ends a step.
// Bound by instruction issue: a step's 32 matrix instructions of a wave take 1024
// cycles of the matrix core but also about 16 each of the issue port that its 260
// vector instructions (a third of them the 2^x and sums of 32 scores a lane) need,
// with two waves per SIMD; the matrix cores are busy for 40% of the time, LDS for
// a quarter. So the steps do without what can be had once: scales sit one block of 16
// keys per lane, and no maximum is taken as long as the weights fit.
//
// Row r of a score tile of 32 keys is the key with bits 2 and 3 of r swapped: a
// lane's scores 8 u .. 8 u + 7 are then the keys 16 u + 8 (lane / 32) .. + 7, the
// operand of the second product's step u. Each such 16 keys lie in one page, so
// their scales are the same in the whole wave.
template <int ST, int DP, bool EXACT, int NW>
__global__ __launch_bounds__(64 * NW, DP <= 128 ? 2 : 1) void k_kv_attend_long(const KvAttendArg a) {
  constexpr int kLongTile = 32 * NW;
  constexpr int NS = DP / 16;          // steps of 16 dimensions in the scores
  constexpr int ND = DP / 32;          // tiles of 32 dimensions
  constexpr int PER = 4 * DP / NW;     // 16-code pieces of a wave and side: a thread's in NL loads
  constexpr int NL = (PER + 63) / 64;
  constexpr bool ALL = PER % 64 == 0;  // every lane has a piece in each
  constexpr int KC = DP / 16;          // 16-code pieces of a key
  constexpr int KR = DP / 8 + 1, VR = kStep / 8 + 1;   // 16-byte chunks of a row in LDS
  const int d = EXACT ? DP : a.d;
  __shared__ u32x4 lk[2][kStep * KR];
  __shared__ u32x4 lv[2][DP * VR];
  __shared__ uint16_t lnan[2][ST == kKvFp8 ? DP * 4 : 1];
  __shared__ int lnan_any[2][NW];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, hf = lane >> 5;

  if (blockIdx.x >= a.tiles) return put_rest(a);
  const int h = blockIdx.x % a.hkv;
  const int rest = blockIdx.x / a.hkv;
  const int split = rest % a.splits;
  const int item = a.items - 1 - rest / a.splits;   // a causal prompt's longest rows first
  const KvTile tl = tile_of(a, item);
  if (tl.b < 0) return;
  const KvSeq s = tl.s;
  const auto [len, bad] = len_of(a, s);
  const int rows = tl.rows, r_first = tl.r_first, n = static_cast<int>(s.n);
  const int r_last = r_first + kLongTile - 1 < rows ? r_first + kLongTile - 1 : rows - 1;
  const int all_hi = keys_of(a, len, n, r_last / a.rep).hi;
  const int kb = keys_of(a, len, n, r_first / a.rep).lo / kStep;
  const int ke = (all_hi + kStep - 1) / kStep;
  const int per = (ke - kb + a.splits - 1) / a.splits;
  const int s0 = kb + split * per;
  const int s1 = s0 + per < ke ? s0 + per : ke;

  // this wave's rows, and this lane's
  const int w_first = r_first + wave * 32;
  const bool w_any = w_first < rows;
  const int w_last = w_first + 31 < rows ? w_first + 31 : rows - 1;
  const KeyRange wf = keys_of(a, len, n, (w_any ? w_first : w_last) / a.rep);
  const KeyRange wl = keys_of(a, len, n, w_last / a.rep);
  const bool has = w_first + n32 < rows;
  const int r = has ? w_first + n32 : rows - 1;
  const int ti = r / a.rep;
  const int head = h * a.rep + r - ti * a.rep;
  const KeyRange mine = keys_of(a, len, n, ti);
  f16x o[ND] = {};
  float m = kNegInf, l = 0.0f, cq;
  u32x4 qf[NS];
  load_q<NS>(a, a.q + (s.tok0 + ti) * a.qts + head * a.qhs, has, [&](int k) { return 16 * k + 8 * hf; },
             [](float v) { return max_halves(v); }, cq, [&](int k) -> u32x4& { return qf[k]; });

  // A step's 64 keys are four blocks of 16 (those past the last are read as the
  // last, masked). Lane l keeps the page id and scales of block l % 4.
  const int last_block = (all_hi - 1) >> 4;
  const int shift = a.m.page_shift;
  const int32_t* trow = a.m.table + tl.b * a.m.tstride;
  auto block_of = [&](int st, int q) {
    const int bl = st * 4 + q;
    return bl < last_block ? bl : last_block;
  };
  auto id_of = [&](int st) { return trow[(block_of(st, lane & 3) << 4) >> shift]; };
  auto known = [&](int id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(a.m.num_pages); };
  u32x4 rk[NL], rv[NL];
  // NW / 4 waves take the keys of each block, all threads the values: lane's block
  // l % 4 of dimension tid / 4.
  const int kblock = wave / (NW / 4), kfirst = (wave % (NW / 4)) * (DP / (NW / 4));
  auto load_codes = [&](int st, int id) {
    id = known(id) ? id : 0;
    const int idk = __builtin_amdgcn_readlane(id, kblock);
    const uint8_t* kp = a.kc + ((static_cast<int64_t>(idk) * a.hkv + h) * a.page +
                                ((block_of(st, kblock) << 4) & (a.page - 1))) * d;
    const uint8_t* vp = a.vc + (static_cast<int64_t>(id) * a.hkv + h) * a.page * d +
                        ((block_of(st, lane & 3) << 4) & (a.page - 1)) + (tid >> 2) * a.page;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int e = kfirst + lane + 64 * i, key = e / KC, dim = 16 * (e % KC);
      const bool here = ALL || lane + 64 * i < PER;
      if (!EXACT || !ALL) rk[i] = u32x4{0, 0, 0, 0};
      if (here && (EXACT || dim < d)) rk[i] = *reinterpret_cast<const u32x4*>(kp + (key * d + dim));
      if (!EXACT || !ALL) rv[i] = u32x4{0, 0, 0, 0};
      if ((EXACT && ALL) || (tid >> 2) + 16 * NW * i < d) rv[i] = *reinterpret_cast<const u32x4*>(vp + 16 * NW * i * a.page);
    }
  };
  // In steps that some row of the workgroup does not see whole, NaN values (FP8)
  // are left out of lv, so that they reach only the rows that see their key (0 x
  // NaN is NaN), and lnan holds a bit for each.
  const int g_hi = keys_of(a, len, n, r_first / a.rep).hi, g_lo = keys_of(a, len, n, r_last / a.rep).lo;
  auto group_masked = [&](int st) { return st * kStep + kStep > g_hi || st * kStep < g_lo; };
  auto nan_in_step = [&](int buf) {
    int any = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) any |= lnan_any[buf][w];
    return __builtin_amdgcn_readfirstlane(any) != 0;
  };
  auto store_codes = [&](int buf, int st) {
    if constexpr (ST == kKvFp8) {
      if (group_masked(st)) {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          uint32_t bits = 0;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t nb = nan_bytes(rv[i][w]) >> 7;
            bits |= (nb * 0x01020408u >> 24 & 0xfu) << (4 * w);   // bytes 0 .. 3 to bits 0 .. 3
            rv[i][w] &= ~(nb * 0xffu);
          }
          if (ALL || (tid >> 2) + 16 * NW * i < DP)
            lnan[buf][((tid >> 2) + 16 * NW * i) * 4 + (lane & 3)] = static_cast<uint16_t>(bits);
          any |= bits;
        }
        const int found = __any(any != 0);
        if (lane == 0) lnan_any[buf][wave] = found;
      }
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int e = kfirst + lane + 64 * i, key = e / KC, dim = 16 * (e % KC);
      if (ALL || lane + 64 * i < PER) {
        u32x4* kp = &lk[buf][(16 * kblock + key) * KR + dim / 8];
        kp[0] = widen8<ST>(rk[i].x, rk[i].y);
        kp[1] = widen8<ST>(rk[i].z, rk[i].w);
      }
      if (ALL || (tid >> 2) + 16 * NW * i < DP) {
        u32x4* vp = &lv[buf][((tid >> 2) + 16 * NW * i) * VR + 2 * (lane & 3)];
        vp[0] = widen8<ST>(rv[i].x, rv[i].y);
        vp[1] = widen8<ST>(rv[i].z, rv[i].w);
      }
    }
  };
  const int krow = (n32 & 0x13) | ((n32 & 4) << 1) | ((n32 & 8) >> 1);

  if (s0 < s1) {
    int id = id_of(s0), id_next = id_of(s0 + 1);     // (steps past the range read its end again, unused)
    load_codes(s0, id);
    auto scale_at = [&](const float* p, int i) { return p[static_cast<int64_t>(known(i) ? i : 0) * a.hkv + h]; };
    float ks = known(id) ? scale_at(a.ks, id) : __builtin_nanf(""), vs = scale_at(a.vs, id);
    store_codes(0, s0);
    load_codes(s0 + 1, id_next);
    id = id_next;
    id_next = id_of(s0 + 2);
    __syncthreads();

    for (int st = s0; st < s1; ++st) {
      const int buf = (st - s0) & 1;
      const int tb = st * kStep;
      // this step's scales, one block of 16 keys per lane; the next ones
      vs = vs < kTinyScale ? kTinyScale : vs;
      const float lane_lvs = __builtin_amdgcn_logf(vs), lane_ivs = __builtin_amdgcn_rcpf(vs);
      float ksq[4], lvs[4], ivs[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        ksq[q] = read_lane(ks, q);
        lvs[q] = read_lane(lane_lvs, q);
        ivs[q] = read_lane(lane_ivs, q);
      }
      ks = known(id) ? scale_at(a.ks, id) : __builtin_nanf("");
      vs = scale_at(a.vs, id);

      if (w_any && tb < wl.hi && tb + kStep > wf.lo) {
        const bool masked = tb + kStep > wf.hi || tb < wl.lo;
        f16x sc[2];
        __builtin_amdgcn_s_setprio(1);   // a wave at its products goes before one at its weights
#pragma unroll
        for (int k = 0; k < NS; ++k)
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) {
            const u32x4 kk = lk[buf][(32 * kt + krow) * KR + 2 * k + hf];
            sc[kt] = mfma32x32x16<kF16>(kk, qf[k], k == 0 ? f16x{} : sc[kt]);
          }
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        // key tb + 16 q + 8 hf + i is outside [lo, hi)
        const int before = mine.lo - tb - 8 * hf;
        const uint32_t wide = static_cast<uint32_t>(mine.hi - mine.lo);
        auto hidden = [&](int q, int i, int from) { return static_cast<uint32_t>(16 * q + i - from) >= wide; };
        // Weights against the maximum so far: as long as none is past fp16's
        // range it stays (their sum tells); else, and at first, it is raised to
        // the step's own and the weights are made again.
        u32x4 p[4];
        float part[4];
        auto weigh = [&](auto mask) {
          const float ref = m == kNegInf ? 0.0f : m;
          const int hide = mask.value ? opaque(before) : 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float f = cq * ksq[q], off = lvs[q] - ref;
            part[q] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float w[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float x = sc[q >> 1][8 * (q & 1) + 2 * i + e];
                w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, f, off));
                if (mask.value && hidden(q, 2 * i + e, hide)) w[e] = 0.0f;   // whatever its scale is
              }
              p[q][i] = pack2_out<kF16>(w[0], w[1]);
              part[q] += w[0] + w[1];   // before their rounding: the sum also counts what is far below
                                        // fp16's range here and large once divided by its scale
            }
          }
        };
        if (masked) weigh(std::true_type{});
        else weigh(std::false_type{});
        const bool needs_here = !((part[0] + part[1]) + (part[2] + part[3]) <= kMostWeight) || m == kNegInf;
        if (__any(needs_here)) {
          // a row whose two lanes need no raising stays as it is, whatever the
          // wave's other rows do
          const bool needs = max_halves(needs_here ? 1.0f : 0.0f) != 0.0f;
          const int hide = opaque(before);
          float mx = kNegInf;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float f = cq * ksq[q];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float y = __builtin_fmaf(sc[q >> 1][8 * (q & 1) + i], f, lvs[q]);
              mx = fmaxf(mx, hidden(q, i, hide) ? kNegInf : y);
            }
          }
          const float top = fmaxf(max_halves(mx), m);
          mx = needs ? top : m;
          const float f = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - mx);
          m = mx;
          l *= f;
#pragma unroll
          for (int t = 0; t < ND; ++t) o[t] *= f;
          weigh(std::true_type{});
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) l += part[q] == 0.0f ? 0.0f : part[q] * ivs[q];
        __builtin_amdgcn_sched_barrier(0);

        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int t = 0; t < ND; ++t)
            o[t] = mfma32x32x16<kF16>(lv[buf][(32 * t + n32) * VR + 2 * q + hf], p[q], o[t]);
        __builtin_amdgcn_s_setprio(0);
        if constexpr (ST == kKvFp8) {
          if (group_masked(st) && nan_in_step(buf)) {
            // the count of NaN values that a row sees in each dimension
            const int hide = opaque(before);
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
              u32x4 seen;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                seen[i] = (hidden(q, 2 * i, hide) ? 0u : 0x3c00u) | (hidden(q, 2 * i + 1, hide) ? 0u : 0x3c000000u);
#pragma unroll
              for (int t = 0; t < ND; ++t) {
                const uint32_t bits = static_cast<uint32_t>(lnan[buf][(32 * t + n32) * 4 + q]) >> (8 * hf);
                u32x4 ind;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  ind[i] = (bits >> (2 * i) & 1u) * 0x3c00u + (bits >> (2 * i + 1) & 1u) * 0x3c000000u;
                const f16x cnt = mfma32x32x16<kF16>(ind, seen, f16x{});
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] += cnt[i] > 0.0f ? __builtin_nanf("") : 0.0f;
              }
            }
          }
        }
      }
      if (st + 1 < s1) {
        store_codes(buf ^ 1, st + 1);
        load_codes(st + 2, id_next);
        id = id_next;
        id_next = id_of(st + 3);
      }
      __syncthreads();
    }
  }
  const float sum = l + __shfl_xor(l, 32, 64);
  if (!has) return;
  const int64_t orow = (s.tok0 + ti) * a.hq + head;
#pragma unroll
  for (int t = 0; t < ND; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d0 = 32 * t + 8 * q + 4 * hf;
      if (EXACT || d0 < d)
        put_row(a, orow, static_cast<int64_t>(item * a.hkv + h) * kLongTile + wave * 32 + n32, split, d0,
                f4{o[t][4 * q], o[t][4 * q + 1], o[t][4 * q + 2], o[t][4 * q + 3]}, m, sum,
                mine.hi <= mine.lo, bad);
    }
}

// Joins the splits' partial results. A wave (WIDE: a workgroup, of whose waves
// each takes every fourth split) per row; lane l reads split l's maximum and sum,
// then all lanes read 4 dimensions of 8 splits at a time. (One split at a time, a
// load behind a load, took 24 us for 64 splits.)
template <bool WIDE>
__global__ __launch_bounds__(kBlock) void k_kv_attend_join(const KvAttendArg a) {
  constexpr int PER = WIDE ? 1 : 4;     // rows of a workgroup
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int parts = a.tile_rows / PER;
  const int row = (blockIdx.x % parts) * PER + (WIDE ? 0 : wave);
  const int rest = blockIdx.x / parts;
  const int h = rest % a.hkv;
  const int item = rest / a.hkv;
  const int64_t prow = static_cast<int64_t>(item * a.hkv + h) * a.tile_rows + row;
  // What is read does not depend on whose row it is (places of rows that are not
  // there exist too): all of it is under way before that is looked up.
  constexpr int STEP = WIDE ? 4 : 1;
  const int d0 = 4 * lane < a.d ? 4 * lane : 0;
  f4 v[8];
  auto load8 = [&](int s0) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int s = s0 + k * STEP < a.splits ? s0 + k * STEP : 0;
      v[k] = *reinterpret_cast<const f4*>(a.po + (s * a.prows + prow) * a.d + d0);
    }
  };
  float2 ml = make_float2(kNegInf, 0.0f);
  if (lane < a.splits) ml = a.pml[lane * a.prows + prow];
  load8(WIDE ? wave : 0);
  const KvTile tl = tile_of(a, item);
  if (tl.b < 0 || tl.r_first + row >= tl.rows) return;
  float m = ml.x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float f = ml.x == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ml.x - m);
  float l = ml.y * f;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o, 64);
  f4 acc = {};
  for (int s0 = WIDE ? wave : 0; s0 < a.splits; s0 += 8 * STEP) {
    if (s0 >= 8 * STEP) load8(s0);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int s = s0 + k * STEP;
      const float fs = s < a.splits ? read_lane(f, s) : 0.0f;   // s is the same in the wave
      if (s < a.splits) acc += v[k] * fs;
    }
  }
  if constexpr (WIDE) {
    __shared__ f4 part[3][64];
    if (wave > 0) part[wave - 1][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < 3; ++w) acc += part[w][lane];
  }
  const int ti = (tl.r_first + row) / a.rep;
  const int64_t orow = (tl.s.tok0 + ti) * a.hq + h * a.rep + (tl.r_first + row - ti * a.rep);
  const auto [len, bad] = len_of(a, tl.s);
  const KeyRange seen = keys_of(a, len, static_cast<int>(tl.s.n), ti);
  KvAttendArg one = a;
  one.splits = 1;
  if (4 * lane < a.d) put_row(one, orow, 0, 0, d0, acc, m, l, seen.hi <= seen.lo, bad);
}

// What one call launches: k_kv_attend_rows for the sequences of few rows,
// k_kv_attend_long for the others (items 0: not launched).
struct KvPlan {
  int64_t row_items, long_items;
  int64_t row_max;         // rows of a sequence that k_kv_attend_rows takes, at most
  int row_splits, long_splits;
  int long_tile;   // rows
};

// Sequences of at most this many rows go to k_kv_attend_rows, and all of them
// where a sequence has at most kFewRows on average, which spares drafted tokens a
// second launch. The mean does not tell of one long sequence among single tokens:
// 255 of those and a chunk of 512, 64 heads over 8 of 128, 8192 keys, take 1045 us in
// this one launch, where the two kernels in calls of their own take 643 and 180 (over
// 2048 keys with 32 heads 228, 166 and 47).
constexpr int64_t kShortRows = 64;
constexpr int64_t kFewRows = 32;
// Where a window leaves every row at most this many keys, and the sequences make at
// most a tile per CU, k_kv_attend_long takes all rows in one launch: a single token's
// tile is then no longer than a prompt's. Measured in one launch and in two, windows
// of 256 / 1024 / 2048 keys, one prompt for every three single tokens:
//   20 sequences, prompts of up to 1500, 4 kv heads of 80   37 / 78 / 131, 49 / 91 / 141 us
//   20, prompts of up to 300, 4 kv heads of 128             40 / 51 / 67,  45 / 56 / 71
//    5, prompts of up to 1500, 4 kv heads of 128            25 / 50 / 82,  38 / 62 / 94
//   32, prompts of up to 600, 8 kv heads of 64              28 / 60 / 101, 28 / 51 / 80
// so what decides is how far the tiles fill the GPU rather than the window: the last,
// with a tile per CU of single tokens alone, loses from 512 keys on.
constexpr int64_t kSharedKeys = 1024;
// Workgroups per CU that the keys of few tiles are split for. 2 fit at once
// (head size 128); with 4 a batch of mixed lengths takes 113 instead of 126 us (64
// sequences of 100 to 8000 tokens), one sequence the same.
constexpr int64_t kRowWgs = 4;
// Workgroups for the tokens of no sequence, in calls with offsets.
constexpr int64_t kRestWgs = 16;

int padded_dim(int d) { return (d + 63) / 64 * 64; }

// Head sizes of k_kv_attend_long: 65 .. 96 in tiles of 96, without a quarter of
// 128's products (a batch with 5 prompts of up to 1500 tokens, head size 80: 91 us,
// padded to 128 95, both in two launches).
int long_dim(int d) { return d > 64 && d <= 96 ? 96 : padded_dim(d); }

// Waves of a k_kv_attend_long workgroup for `rows` rows of each kv head. 8 share a
// step's codes (one workgroup per CU; a prompt of 8192 tokens 588 us, with 4 and two
// workgroups 627), 4 leave less of the GPU idle in the last round of few
// workgroups (a batch with 5 prompts of up to 1500 tokens, in tiles of 128: 105 and 110 us). Other
// head sizes have registers or loads for 4 only.
int long_waves(int dp, int64_t rows, int kv_heads, bool one_sequence) {
  if (dp != 128) return 4;
  const int64_t cus = device_cus(), wgs = cdiv(rows, 256) * kv_heads;
  const bool fills = one_sequence && 10 * wgs >= 9 * cus * cdiv(wgs, cus);
  return fills || wgs >= 3 * cus ? 8 : 4;
}

KvPlan plan_of(const cbq_kv_cache* c, const cbq_kv_batch* b, int rep, int64_t max_length, int64_t window) {
  KvPlan p = {};
  const int64_t rows = b->tokens * rep;
  p.long_tile = 32 * long_waves(long_dim(c->head_dim), rows, c->kv_heads, b->batch == 1);
  if (b->cu == nullptr) {
    p.row_items = b->batch * cdiv(rep, kRowTile);
  } else {
    // n rows make at most n / t + 1 tiles of t
    const bool one = b->batch == 1;
    p.row_max = rows <= kFewRows * b->batch ? rows : kShortRows;
    if (!one || rows <= p.row_max)
      p.row_items = std::min(rows / kRowTile + b->batch, b->batch * cdiv(p.row_max, kRowTile));
    if (rows > p.row_max)
      p.long_items = one ? cdiv(rows, p.long_tile)
                         : rows / p.long_tile + std::min<int64_t>(b->batch, rows / (p.row_max + 1));
    if (p.row_items > 0 && p.long_items > 0 && window > 0 && window <= kSharedKeys &&
        static_cast<int64_t>(b->batch) * c->kv_heads <= device_cus()) {
      p.row_items = 0;
      p.long_items = rows / p.long_tile + std::min<int64_t>(b->batch, rows);
    }
  }
  const int64_t cap = static_cast<int64_t>(b->max_pages) * c->page_size;
  const int64_t len = max_length > 0 ? std::min(max_length, cap) : cap;
  const int64_t cus = device_cus();
  p.row_splits = p.long_splits = 1;
  if (p.row_items > 0) {
    const int64_t want = cdiv(kRowWgs * cus, p.row_items * c->kv_heads);
    p.row_splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, cdiv(cdiv(len, kStep), 4), kMaxSplits})));
  }
  if (p.long_items > 0) {
    const int64_t want = (p.long_tile == 256 ? 1 : 2) * cus / (p.long_items * c->kv_heads);
    p.long_splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, cdiv(len, 8 * kStep), kMaxSplits})));
  }
  return p;
}

size_t partial_bytes(const cbq_kv_cache* c, int64_t items, int tile) {
  return static_cast<size_t>(items) * c->kv_heads * tile * (c->head_dim + 2) * 4;
}

}  // namespace
}  // namespace cbq

using namespace cbq;

extern "C" size_t cbq_kv_attend_ws_bytes(const cbq_kv_cache* cache, const cbq_kv_batch* batch,
                                         int32_t q_heads, int64_t max_length) {
  if (cache == nullptr || batch == nullptr || cache->kv_heads <= 0 || q_heads <= 0 ||
      q_heads % cache->kv_heads != 0 || batch->tokens <= 0)
    return CBQ_WS_CTRL_BYTES;
  const KvPlan p = plan_of(cache, batch, q_heads / cache->kv_heads, max_length, 0);   // (a window's one launch has room for fewer splits, at times)
  size_t n = 0;
  if (p.row_splits > 1) n += p.row_splits * partial_bytes(cache, p.row_items, kRowTile);
  if (p.long_splits > 1) n += p.long_splits * partial_bytes(cache, p.long_items, p.long_tile);
  return CBQ_WS_CTRL_BYTES + n;
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
  CBQ_REQUIRE(batch->tokens * rep < (int64_t{1} << 31) - 512, "kv attend: too many tokens for one call");
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
  a.window = static_cast<int>(std::min<int64_t>(window, INT32_MAX));
  a.negate = scale < 0.0f;
  a.scale_log2e = __builtin_fabsf(scale) * kLog2e;
  a.hkv = cache->kv_heads;
  a.hq = q_heads;
  a.rep = rep;
  a.d = cache->head_dim;
  a.page = cache->page_size;
  a.causal = causal != 0;
  a.bf16 = dtype == CBQ_BF16;
  const KvPlan p = plan_of(cache, batch, rep, max_length, window);
  size_t room = ws != nullptr && ws_bytes > CBQ_WS_CTRL_BYTES ? ws_bytes - CBQ_WS_CTRL_BYTES : 0;
  char* scratch = static_cast<char*>(ws) + CBQ_WS_CTRL_BYTES;
  hipStream_t st = as_stream(stream);
  // One launch over `items` tiles of `tile` rows, the keys in `splits` ranges (as
  // many as the workspace has room for), and the launch that joins them.
  int64_t rest_wgs = batch->cu != nullptr ? kRestWgs : 0;     // in the first launch
  auto run = [&](int64_t items, int tile, int splits, int dim, auto kernel) -> int {
    const size_t each = partial_bytes(cache, items, tile);
    splits = std::max(1, static_cast<int>(std::min<size_t>(splits, room / each)));
    a.items = static_cast<int>(items);
    a.tile_rows = tile;
    a.splits = splits;
    a.prows = items * a.hkv * tile;
    if (splits > 1) {
      a.pml = reinterpret_cast<float2*>(scratch);
      a.po = reinterpret_cast<float*>(a.pml + splits * a.prows);   // 16-byte aligned: prows is even
      scratch += splits * each;
      room -= splits * each;
    }
    const int64_t blocks = items * a.hkv * splits;
    const bool wide = splits > 8;
    const int64_t joins = items * a.hkv * (wide ? tile : tile / 4);
    CBQ_REQUIRE(blocks < (int64_t{1} << 31) - kRestWgs && joins < (int64_t{1} << 31),
                "kv attend: too many tokens for one call");
    a.tiles = static_cast<uint32_t>(blocks);
    const dim3 grid(static_cast<uint32_t>(blocks + rest_wgs));
    rest_wgs = 0;
    auto by_dim = [&](auto stc) {
      switch (dim) {
        case 64: kernel(grid, stc, std::integral_constant<int, 64>{}); break;
        case 96: kernel(grid, stc, std::integral_constant<int, 96>{}); break;
        case 128: kernel(grid, stc, std::integral_constant<int, 128>{}); break;
        case 192: kernel(grid, stc, std::integral_constant<int, 192>{}); break;
        default: kernel(grid, stc, std::integral_constant<int, 256>{}); break;
      }
    };
    if (cache->store == CBQ_KV_INT8) by_dim(std::integral_constant<int, kKvInt8>{});
    else by_dim(std::integral_constant<int, kKvFp8>{});
    if (int rc = launch_status("cbq_kv_attend")) return rc;
    if (splits == 1) return CBQ_OK;
    if (wide) k_kv_attend_join<true><<<dim3(static_cast<uint32_t>(joins)), kBlock, 0, st>>>(a);
    else k_kv_attend_join<false><<<dim3(static_cast<uint32_t>(joins)), kBlock, 0, st>>>(a);
    return launch_status("cbq_kv_attend");
  };
  if (p.row_items > 0) {
    a.row_min = 1;
    a.row_max = batch->cu == nullptr ? rep : static_cast<int>(p.row_max);
    const bool alone = batch->cu == nullptr && rep <= kRowTile;
    const int rc = run(p.row_items, kRowTile, p.row_splits, padded_dim(a.d), [&](dim3 grid, auto stc, auto dpc) {
      constexpr int ST = decltype(stc)::value;
      constexpr int DP = decltype(dpc)::value == 96 ? 128 : decltype(dpc)::value;   // (96 does not come)
      auto go = [&](auto nt) {
        if (a.d == DP) k_kv_attend_rows<ST, DP, true, nt.value><<<grid, kBlock, 0, st>>>(a);
        else k_kv_attend_rows<ST, DP, false, nt.value><<<grid, kBlock, 0, st>>>(a);
      };
      if (alone) go(std::true_type{});
      else go(std::false_type{});
    });
    if (rc) return rc;
  }
  if (p.long_items > 0) {
    a.row_min = p.row_items > 0 ? static_cast<int>(p.row_max) + 1 : 1;
    a.row_max = INT32_MAX;
    return run(p.long_items, p.long_tile, p.long_splits, long_dim(a.d), [&](dim3 grid, auto stc, auto dpc) {
      constexpr int ST = decltype(stc)::value, DP = decltype(dpc)::value;
      auto go = [&](auto nwc) {
        constexpr int NW = decltype(nwc)::value;
        if (a.d == DP) k_kv_attend_long<ST, DP, true, NW><<<grid, 64 * NW, 0, st>>>(a);
        else k_kv_attend_long<ST, DP, false, NW><<<grid, 64 * NW, 0, st>>>(a);
      };
      if constexpr (DP == 128) {
        if (p.long_tile == 256) return go(std::integral_constant<int, 8>{});
      }
      go(std::integral_constant<int, 4>{});
    });
  }
  return CBQ_OK;
}
