// cbq_kv_append.hip - writing and reading back the 8-bit paged key/value cache.
//
// k_kv_append: one workgroup for each (sequence, page that gets new tokens, kv
// head, keys or values), which takes the page's new tokens' maximum, settles
// the page's scale, lowers earlier codes if the scale grew, and writes the new
// codes; and one wave for each new token's queries. A page's head belongs to one
// workgroup, so nothing is atomic and results do not depend on order.
// k_kv_append_step does the same for one new token per sequence.
//
// A thread's unit is 4 tokens x 8 dimensions. Keys: neighbouring lanes take
// neighbouring dimensions (rows of x are read whole, codes written 8 bytes per
// token). Values, stored transposed: neighbouring lanes take neighbouring
// groups of 4 tokens, so that a word of 4 tokens' codes of one dimension is
// made in one thread's registers and stored as it is, without LDS; the 4 lanes
// that share a token still read 64 consecutive bytes of it.
//
// Bound by bytes: the new keys, values and queries in, the queries and codes out.
// Measured on MI355X, kernel times: 8192 tokens of 32 query and 8 kv heads of 128
// (185 MB) 36.8 us, 5.0 TB/s, where a copy reaches 5.1, but 64 with interleaved pairs
// and 126 with a rot_dim that is no multiple of 16 (turned8 for each piece); 256 single
// tokens of 32 and 32 heads of 64 10 us (24 with a workgroup per head); one token 3 us.
// Reading 128 pages of 64 tokens of 8 heads of 128 back (50 MB) 9.8 us, 5.1 TB/s.
#include <algorithm>
#include <type_traits>

#include "cbq_kv.h"

namespace cbq {
namespace {

struct KvHeadsArg {
  const char* p;       // 2-byte elements
  int64_t ts, hs;      // strides in bytes
};

struct KvRopeArg {
  const float* cos;
  const float* sin;
  const int64_t* pos;
  int64_t rows;
  int rot;             // 0: no rotation
  int interleaved;
  int vec;             // whole 8-element pieces can be turned from whole pieces
};

struct KvAppendArg {
  KvBatch m;
  KvHeadsArg k, v, q;
  KvRopeArg rope;
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  char* q_out;
  int64_t kv_blocks;   // k_kv_append: workgroups for pages; the rest are for queries
  int step_waves;      // k_kv_append_step: waves for keys and values; the rest are for queries
  int q_waves;         // waves of a token's queries
  int hkv, hq, d, page;
};

constexpr float kKvEps = 1e-12f;

template <int ST> constexpr float kv_qmax() { return ST == kKvInt8 ? kQmaxInt8 : kQmaxFp8; }

template <int DT>
__device__ __forceinline__ void load8(const char* row, int d0, float (&f)[8]) {
  Raw8<DT> r;
  r.a = ldg16<false>(row + 2 * d0);
  cvt8<DT>(r, f);
}

// Dimensions d0 .. d0 + 7 of one token's head, turned to table row `pos`
// (pos < 0: not a row of the table). Each product and each sum is rounded, so
// the result does not depend on how the pieces are cut.
template <int DT>
__device__ __forceinline__ void turned8(const char* row, int d0, int64_t pos, const KvRopeArg& r,
                                        float (&f)[8]) {
  load8<DT>(row, d0, f);
  if (d0 >= r.rot) return;
  const int half = r.rot >> 1;
  if (pos < 0) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (d0 + k < r.rot) f[k] = __builtin_nanf("");
    return;
  }
  const float* ct = r.cos + pos * half;
  const float* st = r.sin + pos * half;
  if (r.interleaved) {
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      if (d0 + k < r.rot) {
        const int i = (d0 + k) >> 1;
        const float c = ct[i], s = st[i], a = f[k], b = f[k + 1];
        f[k] = a * c - b * s;
        f[k + 1] = b * c + a * s;
      }
    }
  } else if (r.vec) {
    // half is a multiple of 8: the piece and its partners are whole pieces
    const bool first = d0 < half;
    const int i0 = first ? d0 : d0 - half;
    float g[8];
    load8<DT>(row, first ? d0 + half : i0, g);
    const float4 c0 = *reinterpret_cast<const float4*>(ct + i0);
    const float4 c1 = *reinterpret_cast<const float4*>(ct + i0 + 4);
    const float4 s0 = *reinterpret_cast<const float4*>(st + i0);
    const float4 s1 = *reinterpret_cast<const float4*>(st + i0 + 4);
    const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      f[k] = first ? f[k] * c[k] - g[k] * s[k] : f[k] * c[k] + g[k] * s[k];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int e = d0 + k;
      if (e < r.rot) {
        const bool first = e < half;
        const int i = first ? e : e - half;
        const float g = ld1<DT>(row, first ? e + half : i);
        f[k] = first ? f[k] * ct[i] - g * st[i] : f[k] * ct[i] + g * st[i];
      }
    }
  }
}

// Row of the rotation tables for new token `tok` at index `at` of its
// sequence, or -1.
__device__ __forceinline__ int64_t rope_row(const KvRopeArg& r, int64_t tok, int64_t at) {
  const int64_t p = r.pos != nullptr ? r.pos[tok] : at;
  return p >= 0 && p < r.rows ? p : -1;
}

template <int ST>
__device__ __forceinline__ uint2 encode8(const float (&f)[8], float inv) {
  if constexpr (ST == kKvInt8) return pack8_int8(f, inv);
  else return pack8_fp8(f, inv);
}

template <int ST>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float inv) {
  if constexpr (ST == kKvInt8)
    return pack4_low_bytes(q_int8(a * inv), q_int8(b * inv), q_int8(c * inv), q_int8(d * inv));
  else
    return pack4_fp8(a * inv, b * inv, c * inv, d * inv);
}

template <int ST>
__device__ __forceinline__ void decode4(uint32_t w, float* f) {
  if constexpr (ST == kKvInt8) int8x4_to_f32(w, f);
  else fp8x4_to_f32(w, f);
}

// Codes of a word divided by 1 / f (a power of two, or 0), those whose bit in
// `keep` (one byte each) is set left as they are.
template <int ST>
__device__ __forceinline__ uint32_t lower4(uint32_t w, float f, uint32_t keep) {
  float x[4];
  decode4<ST>(w, x);
  const uint32_t n = encode4<ST>(x[0], x[1], x[2], x[3], f);
  return (w & keep) | (n & ~keep);
}

// A page's scale for new tokens of maximum amax: the scale, what new values are
// multiplied by, and what earlier codes are.
struct PageScale {
  float scale, inv, lower;
};

template <int ST>
__device__ __forceinline__ PageScale settle(float amax, float s_old, bool begun) {
  PageScale p;
  if (!begun || s_old == 0.0f) {
    p.inv = inv_scale(amax, kKvEps, kv_qmax<ST>());
    p.scale = 1.0f / p.inv;
    p.lower = 0.0f;         // earlier codes, if any, stand for zeros
    return p;
  }
  p.scale = s_old;
  p.lower = 1.0f;
  float t = amax / (kv_qmax<ST>() * s_old);
  if (t > 1.0f) {
    // A finite maximum may be past fp32's range in units of the smallest scales
    // (a bf16 number above 3.4e26 after zeros): it then grows by 2^64 more than t.
    const bool far = t == __builtin_inff();
    if (far) t = amax * 0x1p-64f / (kv_qmax<ST>() * s_old);
    int e = 0;
    const float mant = __builtin_frexpf(t, &e);
    const int g = (mant > 0.5f ? e : e - 1) + (far ? 64 : 0);
    const bool fin = t < __builtin_inff();
    p.scale = fin ? __builtin_ldexpf(s_old, g) : __builtin_inff();
    p.lower = fin ? __builtin_ldexpf(1.0f, -g) : 0.0f;
  }
  p.inv = 1.0f / p.scale;
  return p;
}

// The first `lo` tokens' codes of a page's head times `lower`, by `n` threads of
// which this is number `i`; 16 codes at a time: of one token (keys) or 16 tokens of
// one dimension (values, of which only the first `lo` change). One load behind the
// other's store, which shows where single tokens make every page grow: 64 tokens of 8
// heads of 128 at the end of their pages 18 us (64 tokens a page) and 77 us (256)
// instead of 4.
template <int ST, bool VALUES>
__device__ void lower_codes(uint8_t* codes, int lo, int page, int d, float lower, int i, int n) {
  if constexpr (VALUES) {
    const int per = page >> 4, used = (lo + 15) >> 4;
    for (int c = i; c < used * d; c += n) {
      const int t0 = (c % used) << 4;
      uint4* p = reinterpret_cast<uint4*>(codes) + (c / used) * per + (t0 >> 4);
      uint4 w = *p;
      uint32_t* q = &w.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int left = lo - t0 - 4 * j;   // tokens of this word to change
        if (left > 0) q[j] = lower4<ST>(q[j], lower, left >= 4 ? 0u : 0xffffffffu << (8 * left));
      }
      *p = w;
    }
  } else {
    for (int c = i; c < lo * d / 16; c += n) {
      uint4* p = reinterpret_cast<uint4*>(codes) + c;
      uint4 w = *p;
      w.x = lower4<ST>(w.x, lower, 0u); w.y = lower4<ST>(w.y, lower, 0u);
      w.z = lower4<ST>(w.z, lower, 0u); w.w = lower4<ST>(w.w, lower, 0u);
      *p = w;
    }
  }
}

// One page, head and side (keys or values).
template <int ST, int DT, bool VALUES>
__device__ void append_page(const KvAppendArg& a, int b, int64_t pnum, int h, float* red) {
  const KvSeq s = kv_seq(a.m, b);
  const int pid = kv_page(a.m, b, pnum);
  if (pid < 0) return;   // the same in every thread of the workgroup
  const int page = a.page, d = a.d;
  const int64_t page0 = pnum << a.m.page_shift;   // index of the page's first token
  const int64_t first = s.len - s.n;              // of the sequence's first new one
  const int lo = static_cast<int>(first > page0 ? first - page0 : 0);
  const int hi = static_cast<int>(s.len - page0 < page ? s.len - page0 : page);
  const KvHeadsArg& src = VALUES ? a.v : a.k;
  const int64_t tokbase = s.tok0 + page0 - first;   // + offset in the page = new token
  const char* x = src.p + h * src.hs;
  const int64_t at = static_cast<int64_t>(pid) * a.hkv + h;
  uint8_t* codes = (VALUES ? a.vc : a.kc) + at * page * d;
  float* scale = (VALUES ? a.vs : a.ks) + at;

  const int tgroups = page >> 2, dgroups = d >> 3, units = tgroups * dgroups;
  auto unit_of = [&](int u, int& t0, int& d0) {
    if constexpr (VALUES) {
      t0 = (u & (tgroups - 1)) << 2;
      d0 = (u / tgroups) << 3;
    } else {
      t0 = (u / dgroups) << 2;
      d0 = (u % dgroups) << 3;
    }
  };
  bool lost = false;   // a token whose position is outside the rotation tables
  // A unit's 4 tokens, those that are not new as the nearest new one (they change
  // no maximum and are not stored): no load waits for another token's branch. (Keys
  // and values of 7527 tokens in pages of 32, 6 heads of 96: 15 us, 18 with a branch
  // per token.)
  auto fetch = [&](int t0, int d0, float (&f)[4][8]) {
    int off[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) off[j] = t0 + j < lo ? lo : t0 + j < hi ? t0 + j : hi - 1;
    if (VALUES || a.rope.rot == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) load8<DT>(x + (tokbase + off[j]) * src.ts, d0, f[j]);
    } else if (a.rope.vec && !a.rope.interleaved && a.rope.rows > 0) {
      const int half = a.rope.rot >> 1;
      const bool turned = d0 < a.rope.rot, low = d0 < half;
      const int i0 = !turned ? 0 : low ? d0 : d0 - half;
      const int dg = !turned ? d0 : low ? d0 + half : i0;
      float g[4][8];
      int64_t pos[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t tok = tokbase + off[j];
        load8<DT>(x + tok * src.ts, d0, f[j]);
        load8<DT>(x + tok * src.ts, dg, g[j]);
        pos[j] = rope_row(a.rope, tok, page0 + off[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool none = pos[j] < 0;
        const int64_t at = (none ? 0 : pos[j]) * half + i0;
        float c[8], sn[8];
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
          *reinterpret_cast<float4*>(c + k) = *reinterpret_cast<const float4*>(a.rope.cos + at + k);
          *reinterpret_cast<float4*>(sn + k) = *reinterpret_cast<const float4*>(a.rope.sin + at + k);
        }
        lost |= none;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float r = f[j][k] * c[k] + g[j][k] * (low ? -sn[k] : sn[k]);
          f[j][k] = !turned ? f[j][k] : none ? __builtin_nanf("") : r;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t tok = tokbase + off[j], pos = rope_row(a.rope, tok, page0 + off[j]);
        lost |= pos < 0;
        turned8<DT>(x + tok * src.ts, d0, pos, a.rope, f[j]);
      }
    }
  };

  float amax = 0.0f;
  float f[4][8] = {};
  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    int t0, d0;
    unit_of(u, t0, d0);
    if (t0 + 4 <= lo || t0 >= hi) continue;
    fetch(t0, d0, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) amax = absmax8(f[j], amax);
  }
  if (lost) amax = __builtin_inff();
  const float s_old = *scale;
  amax = block_max(amax, red);

  const PageScale ps = settle<ST>(amax, s_old, lo > 0);
  const float inv = ps.inv, lower = ps.lower;

  if (lo > 0 && lower != 1.0f) {
    lower_codes<ST, VALUES>(codes, lo, page, d, lower, threadIdx.x, blockDim.x);
    __syncthreads();   // a chunk of values may hold new tokens' places
  }

  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    int t0, d0;
    unit_of(u, t0, d0);
    if (t0 + 4 <= lo || t0 >= hi) continue;
    const bool whole = t0 >= lo && t0 + 4 <= hi;
    if (units > static_cast<int>(blockDim.x)) fetch(t0, d0, f);   // else f still holds the only unit
    if constexpr (VALUES) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        uint8_t* p = codes + (d0 + k) * page + t0;
        const uint32_t w = encode4<ST>(f[0][k], f[1][k], f[2][k], f[3][k], inv);
        if (whole) {
          *reinterpret_cast<uint32_t*>(p) = w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (t0 + j >= lo && t0 + j < hi) p[j] = static_cast<uint8_t>(w >> (8 * j));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (t0 + j >= lo && t0 + j < hi)
          *reinterpret_cast<uint2*>(codes + (t0 + j) * d + d0) = encode8<ST>(f[j], inv);
    }
  }
  if (threadIdx.x == 0) *scale = ps.scale;
}

// The rotated queries of a token, by the wave `wave` of a.q_waves per token. A lane
// keeps one unit, two pieces of 8 dimensions (8 pairs, or 16 that are not rotated),
// of every (64 / units)th head, so the rotation's factors are read once for all of
// them. Interleaved pairs, and pieces that do not fit, go one piece at a time.
template <int DT>
__device__ __forceinline__ void turn_queries(const KvAppendArg& a, int wave) {
  const int tok = wave / a.q_waves, turn = wave % a.q_waves;
  if (tok >= a.m.tokens || a.hq == 0) return;
  int64_t at = -1;
  if (a.m.cu == nullptr) {
    at = static_cast<int64_t>(a.m.lengths[tok]) - 1;
  } else {
    // The token's sequence, by the tokens that each one brings. (One in front of the
    // first sequence's or behind the last's has no position.)
    int rel = 0;
    const int t0 = a.m.cu[0] > 0 ? a.m.cu[0] : 0;
    const int b = tok < t0 ? -1 : kv_find(a.m, tok - t0, rel,
                                          [](const KvSeq& s) { return static_cast<int>(s.n); });
    if (b >= 0) {
      const KvSeq s = kv_seq(a.m, b);
      at = s.len - s.n + rel;
    }
  }
  const int64_t pos = rope_row(a.rope, tok, at);
  const int lane = threadIdx.x & 63;
  const bool two = a.rope.rot == 0 || (a.rope.vec && !a.rope.interleaved && pos >= 0);
  const int units = two ? a.d >> 4 : a.d >> 3, heads = 64 / units;
  const int unit = lane % units;
  const char* x = a.q.p + tok * a.q.ts;
  char* out = a.q_out + static_cast<int64_t>(tok) * a.hq * a.d * 2;
  if (lane >= heads * units) return;
  const int h0 = turn * heads + lane / units, hstep = heads * a.q_waves;
  if (two) {
    const int half = a.rope.rot >> 1;
    const bool turned = 8 * unit < half;
    const int d0 = turned ? 8 * unit : 16 * unit, d1 = turned ? d0 + half : d0 + 8;
    float c[8] = {}, sn[8] = {};
    if (turned) {
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        *reinterpret_cast<float4*>(c + k) = *reinterpret_cast<const float4*>(a.rope.cos + pos * half + d0 + k);
        *reinterpret_cast<float4*>(sn + k) = *reinterpret_cast<const float4*>(a.rope.sin + pos * half + d0 + k);
      }
    }
    for (int h = h0; h < a.hq; h += hstep) {
      float f[8], g[8], o1[8], o2[8];
      load8<DT>(x + h * a.q.hs, d0, f);
      load8<DT>(x + h * a.q.hs, d1, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        o1[k] = turned ? f[k] * c[k] - g[k] * sn[k] : f[k];
        o2[k] = turned ? g[k] * c[k] + f[k] * sn[k] : g[k];
      }
      *reinterpret_cast<uint4*>(out + (static_cast<int64_t>(h) * a.d + d0) * 2) = pack8_out<DT>(o1);
      *reinterpret_cast<uint4*>(out + (static_cast<int64_t>(h) * a.d + d1) * 2) = pack8_out<DT>(o2);
    }
  } else {
    for (int h = h0; h < a.hq; h += hstep) {
      float f[8];
      turned8<DT>(x + h * a.q.hs, 8 * unit, pos, a.rope, f);
      *reinterpret_cast<uint4*>(out + (static_cast<int64_t>(h) * a.d + 8 * unit) * 2) = pack8_out<DT>(f);
    }
  }
}

// Number of pages of a sequence that get new tokens.
struct TouchedPages {
  int shift;
  __device__ int operator()(const KvSeq& s) const {
    const int64_t first = s.len - s.n > 0 ? s.len - s.n : 0;
    if (s.n == 0 || s.len <= first) return 0;
    return static_cast<int>(((s.len - 1) >> shift) - (first >> shift)) + 1;
  }
};

template <int ST, int DT>
__global__ __launch_bounds__(kBlock) void k_kv_append(const KvAppendArg a) {
  __shared__ float red[kBlock / kWave];
  if (blockIdx.x < a.kv_blocks) {
    const int item = blockIdx.x / (2 * a.hkv);
    const int hv = blockIdx.x % (2 * a.hkv);
    int rel = 0;
    const int b = kv_find(a.m, item, rel, TouchedPages{a.m.page_shift});
    if (b < 0) return;
    const KvSeq s = kv_seq(a.m, b);
    const int64_t first = s.len - s.n > 0 ? s.len - s.n : 0;
    const int64_t pnum = (first >> a.m.page_shift) + rel;
    if (hv & 1) append_page<ST, DT, true>(a, b, pnum, hv >> 1, red);
    else append_page<ST, DT, false>(a, b, pnum, hv >> 1, red);
    return;
  }
  turn_queries<DT>(a, (blockIdx.x - a.kv_blocks) * (blockDim.x >> 6) + (threadIdx.x >> 6));
}

// One new token per sequence. A wave takes one side of a token's 64 / LANES kv
// heads, LANES lanes a head, 8 dimensions a lane: where the general kernel has a
// workgroup per head, of which a sixteenth of the lanes have anything to do.
template <int ST, int DT, int LANES, bool VALUES>
__device__ __forceinline__ void append_token(const KvAppendArg& a, int b, int h0) {
  const int lane = threadIdx.x & 63, part = lane % LANES, d0 = 8 * part;
  const int64_t len = a.m.lengths[b], at = len - 1;
  if (len <= 0) return;
  const int pid = kv_page(a.m, b, at >> a.m.page_shift);
  if (pid < 0) return;
  const int off = static_cast<int>(at) & (a.page - 1);
  const int h = h0 + lane / LANES;
  const bool mine = h < a.hkv && d0 < a.d;
  const int64_t place = static_cast<int64_t>(pid) * a.hkv + (h < a.hkv ? h : 0);
  uint8_t* codes = (VALUES ? a.vc : a.kc) + place * a.page * a.d;
  float* scale = (VALUES ? a.vs : a.ks) + place;
  const KvHeadsArg& src = VALUES ? a.v : a.k;
  const float s_old = *scale;
  float f[8] = {};
  bool lost = false;
  if (mine) {
    const char* row = src.p + b * src.ts + h * src.hs;
    if (VALUES || a.rope.rot == 0) {
      load8<DT>(row, d0, f);
    } else {
      const int64_t pos = rope_row(a.rope, b, at);
      lost = pos < 0;
      turned8<DT>(row, d0, pos, a.rope, f);
    }
  }
  float amax = absmax8(f, 0.0f);
  if (lost) amax = __builtin_inff();
  amax = group_max<LANES>(amax);
  const PageScale ps = settle<ST>(amax, s_old, off > 0);
  if (h < a.hkv && off > 0 && ps.lower != 1.0f)
    lower_codes<ST, VALUES>(codes, off, a.page, a.d, ps.lower, part, LANES);
  // a chunk of values may hold the new token's place
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (!mine) return;
  const uint2 w = encode8<ST>(f, ps.inv);
  if constexpr (VALUES) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      codes[(d0 + k) * a.page + off] = static_cast<uint8_t>((k < 4 ? w.x : w.y) >> (8 * (k & 3)));
  } else {
    *reinterpret_cast<uint2*>(codes + off * a.d + d0) = w;
  }
  if (part == 0) *scale = ps.scale;
}

template <int ST, int DT, int LANES>
__global__ __launch_bounds__(kBlock) void k_kv_append_step(const KvAppendArg a) {
  const int wave = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (wave >= a.step_waves) {
    turn_queries<DT>(a, wave - a.step_waves);
    return;
  }
  constexpr int HEADS = 64 / LANES;
  const int per = 2 * ((a.hkv + HEADS - 1) / HEADS);     // waves of a token
  const int b = wave / per, rest = wave % per;
  if (rest & 1) append_token<ST, DT, LANES, true>(a, b, (rest >> 1) * HEADS);
  else append_token<ST, DT, LANES, false>(a, b, (rest >> 1) * HEADS);
}

struct KvDequantArg {
  const uint8_t* kc;
  const uint8_t* vc;
  const float* ks;
  const float* vs;
  const int32_t* pages;
  char* ko;
  char* vo;
  int hkv, d, page, num_pages;
};

// One page, head and side; units and lanes as in append_page.
template <int ST, int OUT>
__global__ __launch_bounds__(kBlock) void k_kv_dequant(const KvDequantArg a) {
  const int64_t item = blockIdx.x / (2 * a.hkv);
  const int hv = blockIdx.x % (2 * a.hkv), h = hv >> 1;
  const bool values = hv & 1;
  const int id = a.pages[item];
  const bool ok = static_cast<uint32_t>(id) < static_cast<uint32_t>(a.num_pages);
  const int64_t at = static_cast<int64_t>(ok ? id : 0) * a.hkv + h;
  const uint8_t* codes = (values ? a.vc : a.kc) + at * a.page * a.d;
  const float s = ok ? (values ? a.vs : a.ks)[at] : __builtin_nanf("");
  char* out = (values ? a.vo : a.ko) + (item * a.hkv + h) * a.page * a.d * 2;
  const int tgroups = a.page >> 2, dgroups = a.d >> 3;
  for (int u = threadIdx.x; u < tgroups * dgroups; u += blockDim.x) {
    float f[4][8];
    int t0, d0;
    if (values) {
      t0 = (u & (tgroups - 1)) << 2;
      d0 = (u / tgroups) << 3;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float x[4];
        decode4<ST>(*reinterpret_cast<const uint32_t*>(codes + (d0 + k) * a.page + t0), x);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j][k] = x[j];
      }
    } else {
      t0 = (u / dgroups) << 2;
      d0 = (u % dgroups) << 3;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint2 w = *reinterpret_cast<const uint2*>(codes + (t0 + j) * a.d + d0);
        decode4<ST>(w.x, f[j]);
        decode4<ST>(w.y, f[j] + 4);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        f[j][k] *= s;
        asm volatile("" : "+v"(f[j][k]));   // a finished fp32 product, as in out1
      }
      *reinterpret_cast<uint4*>(out + ((t0 + j) * a.d + d0) * 2) = pack8_out<OUT>(f[j]);
    }
  }
}

// Threads that have a unit to work on, in whole waves.
int block_for(int units) {
  return units >= kBlock ? kBlock : static_cast<int>(cdiv(units, kWave)) * kWave;
}

}  // namespace

int kv_check_cache(const cbq_kv_cache* c) {
  CBQ_REQUIRE(c != nullptr, "kv cache: null cache");
  CBQ_REQUIRE(c->store == CBQ_KV_INT8 || c->store == CBQ_KV_FP8,
              "kv cache: store must be CBQ_KV_INT8 or CBQ_KV_FP8, got %d", c->store);
  CBQ_REQUIRE(c->head_dim >= 16 && c->head_dim <= 256 && c->head_dim % 16 == 0,
              "kv cache: head_dim must be a multiple of 16 in [16, 256], got %d", c->head_dim);
  CBQ_REQUIRE(c->page_size >= 16 && c->page_size <= 256 && (c->page_size & (c->page_size - 1)) == 0,
              "kv cache: page_size must be 16, 32, 64, 128 or 256, got %d", c->page_size);
  CBQ_REQUIRE(c->kv_heads > 0 && c->kv_heads <= 65535, "kv cache: kv_heads must be in [1, 65535], got %d",
              c->kv_heads);
  CBQ_REQUIRE(c->num_pages >= 0 && c->num_pages < (int64_t{1} << 31),
              "kv cache: num_pages must be in [0, 2^31), got %lld", (long long)c->num_pages);
  if (c->num_pages > 0) {
    CBQ_REQUIRE(c->k && c->v && c->k_scale && c->v_scale, "kv cache: null pointer");
    CBQ_REQUIRE(aligned(c->k, 16) && aligned(c->v, 16), "kv cache: codes must be 16-byte aligned");
  }
  return CBQ_OK;
}

int kv_check_batch(const cbq_kv_batch* b) {
  CBQ_REQUIRE(b != nullptr, "kv batch: null batch");
  CBQ_REQUIRE(b->batch >= 0 && b->tokens >= 0 && b->max_pages >= 0, "kv batch: negative size");
  CBQ_REQUIRE(b->cu != nullptr || b->tokens == b->batch,
              "kv batch: without cu there is one new token per sequence, got %lld tokens of %d",
              (long long)b->tokens, b->batch);
  CBQ_REQUIRE(b->tokens < (int64_t{1} << 31), "kv batch: too many tokens");
  if (b->batch > 0 && b->tokens > 0) {
    CBQ_REQUIRE(b->lengths != nullptr, "kv batch: null lengths");
    CBQ_REQUIRE(b->max_pages == 0 || b->page_table != nullptr, "kv batch: null page_table");
    CBQ_REQUIRE(b->table_stride >= b->max_pages, "kv batch: table_stride below max_pages");
  }
  return CBQ_OK;
}

int kv_check_heads(const char* name, const cbq_kv_heads* h) {
  CBQ_REQUIRE(h != nullptr && h->data != nullptr, "kv: null %s", name);
  CBQ_REQUIRE(aligned(h->data, 16) && h->token_stride % 8 == 0 && h->head_stride % 8 == 0,
              "kv: %s must be 16-byte aligned with strides that are multiples of 8 elements", name);
  return CBQ_OK;
}

KvBatch kv_batch_of(const cbq_kv_cache* c, const cbq_kv_batch* b) {
  KvBatch m;
  m.table = b->page_table;
  m.lengths = b->lengths;
  m.cu = b->cu;
  m.tstride = b->table_stride;
  m.tokens = b->tokens;
  m.batch = b->batch;
  m.max_pages = b->max_pages;
  m.page_shift = __builtin_ctz(static_cast<unsigned>(c->page_size));
  m.num_pages = static_cast<int>(c->num_pages);
  return m;
}

}  // namespace cbq

using namespace cbq;

extern "C" int cbq_kv_append(const cbq_kv_cache* cache, const cbq_kv_batch* batch, int dtype,
                             const cbq_kv_heads* k, const cbq_kv_heads* v, const cbq_kv_heads* q,
                             int32_t q_heads, const cbq_kv_rope* rope, void* q_out,
                             cbq_stream_t stream) {
  clear_error();
  if (int rc = kv_check_cache(cache)) return rc;
  if (int rc = kv_check_batch(batch)) return rc;
  CBQ_REQUIRE(dtype == CBQ_F16 || dtype == CBQ_BF16, "kv append: dtype must be fp16 or bf16, got %d",
              dtype);
  CBQ_REQUIRE(q_heads >= 0, "kv append: q_heads must not be negative, got %d", q_heads);
  const bool has_q = q != nullptr && q->data != nullptr && q_heads > 0;
  KvRopeArg r = {};
  if (rope != nullptr && rope->rot_dim != 0) {
    CBQ_REQUIRE(rope->rot_dim > 0 && rope->rot_dim % 2 == 0 && rope->rot_dim <= cache->head_dim,
                "kv append: rot_dim must be even and at most head_dim %d, got %d", cache->head_dim,
                rope->rot_dim);
    CBQ_REQUIRE(rope->rows >= 0, "kv append: negative rows of the rotation tables");
    CBQ_REQUIRE(rope->rows == 0 || (rope->cos_table && rope->sin_table),
                "kv append: null rotation table");
    CBQ_REQUIRE(aligned(rope->cos_table, 16) && aligned(rope->sin_table, 16),
                "kv append: rotation tables must be 16-byte aligned");
    r.cos = rope->cos_table;
    r.sin = rope->sin_table;
    r.pos = rope->positions;
    r.rows = rope->rows;
    r.rot = rope->rot_dim;
    r.interleaved = rope->interleaved != 0;
    r.vec = rope->rot_dim % 16 == 0;
  }
  if (batch->tokens == 0 || batch->batch == 0) return CBQ_OK;
  if (int rc = kv_check_heads("k", k)) return rc;
  if (int rc = kv_check_heads("v", v)) return rc;
  if (has_q) {
    if (int rc = kv_check_heads("q", q)) return rc;
    CBQ_REQUIRE(q_out != nullptr && aligned(q_out, 16), "kv append: q_out must be given, 16-byte aligned");
  }
  KvAppendArg a = {};
  a.m = kv_batch_of(cache, batch);
  auto heads = [](const cbq_kv_heads* h) {
    return KvHeadsArg{static_cast<const char*>(h->data), 2 * h->token_stride, 2 * h->head_stride};
  };
  a.k = heads(k);
  a.v = heads(v);
  if (has_q) a.q = heads(q);
  a.rope = r;
  a.kc = static_cast<uint8_t*>(cache->k);
  a.vc = static_cast<uint8_t*>(cache->v);
  a.ks = cache->k_scale;
  a.vs = cache->v_scale;
  a.q_out = static_cast<char*>(q_out);
  a.hkv = cache->kv_heads;
  a.hq = has_q ? q_heads : 0;
  a.d = cache->head_dim;
  a.page = cache->page_size;
  const int64_t T = batch->tokens, B = batch->batch;
  hipStream_t st = as_stream(stream);
  // few tokens: their queries over more waves
  a.q_waves = T <= 1024 ? 4 : 1;
  const bool f16 = dtype == CBQ_F16;
  auto by_type = [&](auto kernel) {
    if (cache->store == CBQ_KV_INT8) {
      if (f16) kernel(std::integral_constant<int, kKvInt8>{}, std::integral_constant<int, kF16>{});
      else kernel(std::integral_constant<int, kKvInt8>{}, std::integral_constant<int, kBF16>{});
    } else {
      if (f16) kernel(std::integral_constant<int, kKvFp8>{}, std::integral_constant<int, kF16>{});
      else kernel(std::integral_constant<int, kKvFp8>{}, std::integral_constant<int, kBF16>{});
    }
  };
  const int64_t q_total = has_q ? T * a.q_waves : 0;
  if (batch->cu == nullptr) {
    const int lanes = a.d <= 64 ? 8 : a.d <= 128 ? 16 : 32;
    const int64_t waves = B * 2 * cdiv(a.hkv, 64 / lanes);
    CBQ_REQUIRE(waves + q_total < (int64_t{1} << 31) - 4, "kv append: too many tokens for one call");
    a.step_waves = static_cast<int>(waves);
    const dim3 grid(static_cast<uint32_t>(cdiv(waves + q_total, 4)));
    by_type([&](auto stc, auto dtc) {
      constexpr int ST = decltype(stc)::value, DT = decltype(dtc)::value;
      if (lanes == 8) k_kv_append_step<ST, DT, 8><<<grid, kBlock, 0, st>>>(a);
      else if (lanes == 16) k_kv_append_step<ST, DT, 16><<<grid, kBlock, 0, st>>>(a);
      else k_kv_append_step<ST, DT, 32><<<grid, kBlock, 0, st>>>(a);
    });
    return launch_status("cbq_kv_append");
  }
  // n new tokens touch at most n pages and at most n / page + 2
  const int64_t pages = std::min(T / a.page + 2 * B, T);
  const int threads = block_for(a.page * a.d / 32);
  a.kv_blocks = pages * 2 * a.hkv;
  const int64_t blocks = a.kv_blocks + cdiv(q_total, threads / 64);
  CBQ_REQUIRE(blocks < (int64_t{1} << 31) && q_total < (int64_t{1} << 31) - 4,
              "kv append: too many tokens for one call");
  const dim3 grid(static_cast<uint32_t>(blocks));
  by_type([&](auto stc, auto dtc) {
    k_kv_append<decltype(stc)::value, decltype(dtc)::value><<<grid, threads, 0, st>>>(a);
  });
  return launch_status("cbq_kv_append");
}

extern "C" int cbq_kv_dequant(const cbq_kv_cache* cache, const int32_t* pages, int64_t n,
                              void* k_out, void* v_out, int out_dtype, cbq_stream_t stream) {
  clear_error();
  if (int rc = kv_check_cache(cache)) return rc;
  CBQ_REQUIRE(out_dtype == CBQ_F16 || out_dtype == CBQ_BF16,
              "kv dequant: out_dtype must be fp16 or bf16, got %d", out_dtype);
  CBQ_REQUIRE(n >= 0, "kv dequant: negative number of pages");
  if (n == 0) return CBQ_OK;
  CBQ_REQUIRE(pages && k_out && v_out, "kv dequant: null pointer");
  CBQ_REQUIRE(aligned(k_out, 16) && aligned(v_out, 16), "kv dequant: outputs must be 16-byte aligned");
  CBQ_REQUIRE(cache->num_pages > 0, "kv dequant: the cache has no pages");
  const int64_t blocks = n * 2 * cache->kv_heads;
  CBQ_REQUIRE(blocks < (int64_t{1} << 31), "kv dequant: too many pages for one call");
  KvDequantArg a;
  a.kc = static_cast<const uint8_t*>(cache->k);
  a.vc = static_cast<const uint8_t*>(cache->v);
  a.ks = cache->k_scale;
  a.vs = cache->v_scale;
  a.pages = pages;
  a.ko = static_cast<char*>(k_out);
  a.vo = static_cast<char*>(v_out);
  a.hkv = cache->kv_heads;
  a.d = cache->head_dim;
  a.page = cache->page_size;
  a.num_pages = static_cast<int>(cache->num_pages);
  const int threads = block_for(a.page * a.d / 32);
  const dim3 grid(static_cast<uint32_t>(blocks));
  hipStream_t st = as_stream(stream);
  const bool f16 = out_dtype == CBQ_F16;
  if (cache->store == CBQ_KV_INT8) {
    if (f16) k_kv_dequant<kKvInt8, kF16><<<grid, threads, 0, st>>>(a);
    else k_kv_dequant<kKvInt8, kBF16><<<grid, threads, 0, st>>>(a);
  } else {
    if (f16) k_kv_dequant<kKvFp8, kF16><<<grid, threads, 0, st>>>(a);
    else k_kv_dequant<kKvFp8, kBF16><<<grid, threads, 0, st>>>(a);
  }
  return launch_status("cbq_kv_dequant");
}
