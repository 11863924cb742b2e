// cbq_w8a8.hip - products of INT8 activations and INT8 weights with a scale for
// each token and output channel, on gfx950 matrix cores, and the first half of a
// gated block: both projections, the activation and their product in one kernel.
//
//   y[m, n] = sx[m] sw[n] sum_k x[m, k] w[n, k] + bias[n]
//   y[m, n] = act(g) u,  g and u as above with the gate's and the up rows
//
// Sums are int32 and exact (K <= 131071). M <= 64, and products of up to kFewRows rows where its
// model is the faster one: cbq_w8a8_few.hip.
//
// k_w8_tile<J, I, NS, ACT, SPLIT, ANY>: tiles of 64 J tokens x 64 I weight rows (gated:
// 32 I columns of each projection side by side, so that a lane holds g and u of the
// same outputs) of v_mfma_i32_32x32x32_i8, 4 waves of 32 J x 32 I. k-steps of 128 bytes,
// a cache line of every row (steps of 64 asked the L2 for each line twice); NS LDS
// stages filled by LDS DMA; one barrier per k-step, in front of its last quarter.
//
// LDS layout of a stage: the tile's rows of x, then its weight rows, 128 bytes each;
// 16-byte chunk c of row r at c ^ (r / 2 & 7): no bank conflicts, where c ^ (r & 7) cost a
// read 8 cycles instead of 4 (at the same time: the reads hide behind the products). In
// quarter s of a k-step the lanes of half h (lane / 32) take chunk 2 s + h of both operands.
//
// A = weight rows, B = activation rows: lane l holds the outputs of token m = l % 32
// and n = 8 (v / 4) + 4 (l / 32) + v % 4. Outputs leave through LDS, 32 tokens at a
// time per wave, and are stored 16 bytes per lane along a row.
//
// ANY: rows that are no multiples of 16 bytes, which the DMA does not take. They pass
// through registers, loaded a k-step ahead: a k-step of 128 x 128 takes 0.9 us where rows
// are whole words and 1.2 where not, instead of 0.6 (loads from the multiple of 4 in
// front, shifted by the vector unit: 1.7). Many tokens: k_w8_pad.
//
// K is cut into ranges where few tiles would leave CUs idle: each range writes its
// sums to the workspace and k_w8_join adds them (integers: exact in any order).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cbq_lds_dma.h"
#include "cbq_w8a8.h"

namespace cbq {
namespace {

template <int J, int I, int NS> struct W8Geom {
  static constexpr int kWaves = 4;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kTM = 64 * J, kTN = 64 * I;      // rows of x, weight rows
  static constexpr int kX = kTM * 128;                  // bytes of x per stage
  static constexpr int kSB = (kTM + kTN) * 128;
  static constexpr int kLX = 2 * J, kLW = 2 * I;        // loads per thread and stage
  static constexpr int kPitch = 128 * I + 16;           // row of outputs in LDS, bytes
  static_assert(kWaves * 32 * kPitch <= NS * kSB, "the outputs fit in the stages");
  static_assert((NS - 1) * (kLX + kLW) <= 63, "loads in flight are counted in 6 bits");
};

// Workgroup -> (tile m, tile n): XCD b % 8 takes a contiguous run of tiles, in
// groups of 8 tile rows, so that what runs on an XCD shares rows in its L2.
__device__ __forceinline__ void w8_tile(int b, const W8Args& a, int& tm, int& tn) {
  const int total = a.tiles_m * a.tiles_n;
  b = static_cast<int>(xcd_remap(b, total));
  constexpr int G = 8;
  const int group = b / (G * a.tiles_n);
  const int first_m = group * G;
  const int gsize = min(a.tiles_m - first_m, G);
  const int r = b % (G * a.tiles_n);
  tm = first_m + r % gsize;
  tn = r / gsize;
}

template <int J, int I, int NS, int ACT, bool SPLIT, bool ANY>
__global__ __launch_bounds__(256) void k_w8_tile(W8Args a) {
  typedef W8Geom<J, I, NS> G;
  constexpr bool GATED = ACT != kNoAct;
  static_assert(!GATED || I % 2 == 0, "pairs of tiles");
  static_assert(!ANY || NS == 2, "two stages");
  constexpr int LX = G::kLX, LT = G::kLX + G::kLW, NW = G::kWaves;
  constexpr int WM = 32 * J, WR = 32 * I;               // a wave's tokens, weight rows
  constexpr int WN = GATED ? WR / 2 : WR;               // and output columns
  __shared__ __attribute__((aligned(1024))) uint8_t smem[NS * G::kSB];
  __shared__ __attribute__((aligned(16))) float s_x[G::kTM], s_w[G::kTN], s_b[G::kTN];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int r32 = lane & 31, h = lane >> 5;
  const int tiles = a.tiles_m * a.tiles_n;
  const int split = SPLIT ? blockIdx.x / tiles : 0;
  int tm, tn;
  w8_tile(SPLIT ? blockIdx.x % tiles : blockIdx.x, a, tm, tn);
  const int m0 = tm * G::kTM, n0 = tn * 2 * WN;
  const int steps = (a.K + 127) >> 7;
  const int kb = split * a.split_steps;                 // first k-step of this range
  const int nk = SPLIT ? min(a.split_steps, steps - kb) : steps;
  const uint32_t sbase = __builtin_amdgcn_readfirstlane(lds_addr(smem));

  // Weight row r of the tile: its projection, and its column from n0 on. Gated: a
  // wave's rows are WN of the gate, then the same WN of the up projection.
  auto proj_of = [&](int r) { return GATED ? (r % WR) / WN : 0; };
  auto col_of = [&](int r) { return GATED ? r / WR * WN + r % WN : r; };

  if constexpr (!SPLIT) {   // scales and biases of the tile's rows and columns
    for (int r = tid; r < G::kTM; r += 256) s_x[r] = a.sx[min(m0 + r, a.M - 1) * a.sx_step];
    for (int r = tid; r < G::kTN; r += 256) {
      const int p = proj_of(r);
      const int64_t n = min(n0 + col_of(r), a.N - 1);
      s_w[r] = p ? a.sw[1][n * a.sw_step[1]] : a.sw[0][n * a.sw_step[0]];
      const void* b = p ? a.bias[1] : a.bias[0];
      s_b[r] = b ? ld_any(b, a.bias_dt, n) : 0.0f;
    }
  }

  // Load u of a stage: rows (u NW + wave) 8 + lane / 8 (of x, then of the weight), the
  // chunk that belongs at slot lane % 8. Rows past M or N are the last row's; their
  // products are not stored. Chunks past K are the last one's (ANY: see there); x counts
  // as zero there.
  const int lrow = lane >> 3;
  const int lk = ((lane & 7) ^ (((wave & 1) << 2) | (lrow >> 1))) << 4;
  uint32_t off[LT];                                     // of the row, from its base
  const uint8_t* base[LT];
#pragma unroll
  for (int u = 0; u < LT; ++u) {
    if (u < LX) {
      const int r = (u * NW + wave) * 8 + lrow;
      off[u] = static_cast<uint32_t>(min(r, a.M - 1 - m0)) * static_cast<uint32_t>(a.ldx);
      base[u] = a.x + m0 * a.ldx;
    } else {
      const int r = ((u - LX) * NW + wave) * 8 + lrow;
      const int p = __builtin_amdgcn_readfirstlane(proj_of(r));
      off[u] = static_cast<uint32_t>(min(col_of(r), a.N - 1 - n0)) *
               static_cast<uint32_t>(p ? a.ldw[1] : a.ldw[0]);
      base[u] = p ? a.w[1] + n0 * a.ldw[1] : a.w[0] + n0 * a.ldw[0];
    }
  }
  auto issue_one = [&](int t, int u) {                  // t: k-step of this range
    const int k = min((kb + t) * 128 + lk, a.K - 16);
    if constexpr (!ANY)
      lds_dma16(off[u] + static_cast<uint32_t>(k), uniform_ptr(base[u]),
                sbase + (t % NS) * G::kSB + (u < LX ? 0 : G::kX) + ((u < LX ? u : u - LX) * NW + wave) * 1024);
  };
  u32x4 held[ANY ? LT : 1];                             // ANY: a tile's loads on their way to LDS
  auto hold_one = [&](int t, int u) { held[u] = ld_codes(base[u] + off[u], (kb + t) * 128 + lk, a.K); };
  auto land = [&](int t, int u) {
    u32x4 v = held[u];
    if ((kb + t) * 128 + 128 > a.K) v = from_k(v, (kb + t) * 128 + lk, a.K);
    *reinterpret_cast<u32x4*>(smem + (t % NS) * G::kSB + (u < LX ? 0 : G::kX) +
                              ((u < LX ? u : u - LX) * NW + wave) * 1024 + lane * 16) = v;
  };

  const uint32_t xr = (wm * WM + r32) * 128, wr = G::kX + (wn * WR + r32) * 128;
  uint32_t slot[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) slot[s] = static_cast<uint32_t>((2 * s + h) ^ (r32 >> 1 & 7)) << 4;
  i16x acc[J][I];          // [token tile][weight tile]
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < I; ++i) acc[j][i] = i16x{};
  struct Frags { i4v x[J], w[I]; };
  auto read_one = [&](int t, int s, Frags& f, int r) {  // fragment r of quarter s
    const uint8_t* st = smem + (t % NS) * G::kSB;
    if (r < I) f.w[r] = *reinterpret_cast<const i4v*>(st + wr + slot[s] + r * 4096);
    else f.x[r - I] = *reinterpret_cast<const i4v*>(st + xr + slot[s] + (r - I) * 4096);
  };
  // The products of one quarter, with n pieces of other work spread between them.
  auto quarter = [&](const Frags& f, auto n, auto&& work) {
#pragma unroll
    for (int q = 0; q < J * I; ++q) {
      acc[q / I][q % I] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[q % I], f.x[q / I], acc[q / I][q % I],
                                                                0, 0, 0);
#pragma unroll
      for (int e = decltype(n)::value * q / (J * I); e < decltype(n)::value * (q + 1) / (J * I); ++e) work(e);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr std::integral_constant<int, J + I> kReads{};
  constexpr std::integral_constant<int, J + I + LT> kAll{};

  // Step t: the products of a quarter run with the reads of the next one between them.
  // In front of the last quarter every fragment of tile t is read and, past the wait
  // and the barrier, tile t + 1 is there: its stage is read from and tile t + NS takes
  // tile t's. more: there is a tile t + NS; all: wait for every load in flight.
  Frags f0, f1;
  auto step = [&](int t, auto more, auto all) {
    quarter(f0, kReads, [&](int e) { read_one(t, 1, f1, e); });
    quarter(f1, kReads, [&](int e) { read_one(t, 2, f0, e); });
    quarter(f0, kReads, [&](int e) { read_one(t, 3, f1, e); });
    dma_wait_barrier<decltype(all)::value ? 0 : (NS - 2) * LT>();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (decltype(more)::value)
      quarter(f1, kAll, [&](int e) {
        if (e < J + I) read_one(t + 1, 0, f0, e);
        else issue_one(t + NS, e - J - I);
      });
    else quarter(f1, kReads, [&](int e) { read_one(t + 1, 0, f0, e); });
  };
  // ANY: tile t + 1 lands during the third quarter, and its registers are loaded again
  // (past the end with some chunk that is not used).
  auto step_any = [&](int t) {
    quarter(f0, kReads, [&](int e) { read_one(t, 1, f1, e); });
    quarter(f1, kReads, [&](int e) { read_one(t, 2, f0, e); });
    quarter(f0, kAll, [&](int e) {
      if (e < J + I) read_one(t, 3, f1, e);
      else land(t + 1, e - J - I);
    });
    __syncthreads();
    quarter(f1, kAll, [&](int e) {
      if (e < J + I) read_one(t + 1, 0, f0, e);
      else hold_one(t + 2, e - J - I);
    });
  };
  using yes = std::true_type;
  using no = std::false_type;
  if constexpr (ANY) {
#pragma unroll
    for (int u = 0; u < LT; ++u) hold_one(0, u);
#pragma unroll
    for (int u = 0; u < LT; ++u) land(0, u);
#pragma unroll
    for (int u = 0; u < LT; ++u) hold_one(1, u);
    __syncthreads();
  } else {
#pragma unroll
    for (int t = 0; t < NS; ++t)
      if (t < nk) {
#pragma unroll
        for (int u = 0; u < LT; ++u) issue_one(t, u);
      }
    if (nk >= NS) dma_wait_barrier<(NS - 1) * LT>();
    else dma_wait_barrier<0>();
  }
#pragma unroll
  for (int r = 0; r < J + I; ++r) read_one(0, 0, f0, r);
  int t = 0;
  if constexpr (ANY) {
    for (; t + 1 < nk; ++t) step_any(t);
  } else {
    for (; t + NS < nk; ++t) step(t, yes{}, no{});
    for (; t + 1 < nk; ++t) step(t, no{}, yes{});
  }
  // The last tile. Where K ends inside it, x is zero from there on.
  auto cut = [&](Frags& f, int s) {
    if (!ANY && (kb + t) * 128 + (2 * s + h) * 16 >= a.K) {
#pragma unroll
      for (int j = 0; j < J; ++j) f.x[j] = i4v{0, 0, 0, 0};
    }
  };
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    Frags& now = s & 1 ? f1 : f0;
    Frags& next = s & 1 ? f0 : f1;
    cut(now, s);
    quarter(now, kReads, [&](int e) {
      if (s < 3) read_one(t, s + 1, next, e);
    });
  }

  // A range's sums go to the workspace as they lie in registers, 1 KiB per store.
  if constexpr (SPLIT) {
    i4v* dst = reinterpret_cast<i4v*>(a.part) +
               ((static_cast<int64_t>(split) * tiles + tm * a.tiles_n + tn) * NW + wave) * (J * I * 256) + lane;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          __builtin_nontemporal_store(
              i4v{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]},
              dst + ((j * I + i) * 4 + q) * 64);
    return;
  }

  // Outputs: the sums of 32 tokens at a time go through the wave's own part of LDS as
  // they are (straight from the accumulation registers, which the vector unit cannot
  // read) and are finished on the other side, where a lane keeps its columns, and with
  // them their scales, for all rows.
  __syncthreads();
  uint8_t* const out = smem + wave * 32 * G::kPitch;
  const int mw = m0 + wm * WM, nw = n0 + wn * WN;       // the wave's first token and column
  const float* const cols = s_w + wn * WR;              // gated: the up projection's WN further
  const float* const bias = s_b + wn * WR;
  auto finish = [&](int sum, int sum2, float sx, float w0, float b0, float w1, float b1) {
    const float v = scaled(sum, sx, w0, b0);
    return GATED ? activate<ACT>(v) * scaled(sum2, sx, w1, b1) : v;
  };
  // C columns per lane and row: st(row, column, values). ROLL keeps the rows in a loop.
  auto put = [&](auto per_lane, auto roll, auto&& st) {
    constexpr int C = decltype(per_lane)::value, LR = WN / C, RL = 64 / LR;   // lanes of a row, rows at a time
    constexpr int kUnroll = decltype(roll)::value ? 1 : 32 / RL;
    const int c = lane % LR * C;
    float w0[C], b0[C], w1[C], b1[C];
#pragma unroll
    for (int e = 0; e < C; ++e) {
      w0[e] = cols[c + e];
      b0[e] = bias[c + e];
      w1[e] = GATED ? cols[WN + c + e] : 0.0f;
      b1[e] = GATED ? bias[WN + c + e] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      wave_lds_fence();                                 // the last rows are read
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<i4v*>(out + r32 * G::kPitch + (32 * i + 8 * q + 4 * h) * 4) =
              i4v{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
      wave_lds_fence();                                 // written before it is read
#pragma unroll kUnroll
      for (int r = 0; r < 32 / RL; ++r) {
        const int row = r * RL + lane / LR;
        const uint8_t* src = out + row * G::kPitch + c * 4;
        const float sx = s_x[wm * WM + 32 * j + row];
        float v[C];
#pragma unroll
        for (int e = 0; e < C; e += 4) {
          const i4v g = *reinterpret_cast<const i4v*>(src + e * 4);
          i4v u = {0, 0, 0, 0};
          if constexpr (GATED) u = *reinterpret_cast<const i4v*>(src + WN * 4 + e * 4);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[e + k] = finish(g[k], u[k], sx, w0[e + k], b0[e + k], w1[e + k], b1[e + k]);
        }
        if (mw + 32 * j + row < a.M) st(mw + 32 * j + row, nw + c, v);
      }
    }
  };
  auto put16 = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    put(std::integral_constant<int, 8>{}, std::false_type{}, [&](int m, int n, const float (&v)[8]) {
      if (n < a.N)
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.y) + static_cast<int64_t>(m) * a.N + n) =
            u32x4{pack2_out<DT>(v[0], v[1]), pack2_out<DT>(v[2], v[3]), pack2_out<DT>(v[4], v[5]),
                  pack2_out<DT>(v[6], v[7])};
    });
  };
  if (a.vec && a.out_dt == kF16) put16(std::integral_constant<int, kF16>{});
  else if (a.vec && a.out_dt == kBF16) put16(std::integral_constant<int, kBF16>{});
  else if (a.vec)
    put(std::integral_constant<int, 4>{}, std::false_type{}, [&](int m, int n, const float (&v)[4]) {
      if (n < a.N)
        *reinterpret_cast<f4v*>(static_cast<float*>(a.y) + static_cast<int64_t>(m) * a.N + n) =
            f4v{v[0], v[1], v[2], v[3]};
    });
  else
    put(std::integral_constant<int, 4>{}, std::true_type{}, [&](int m, int n, const float (&v)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < a.N) st_any(a.y, a.out_dt, static_cast<int64_t>(m) * a.N + n + e, v[e]);
    });
}

// Adds the ranges' sums and finishes the outputs. A workgroup has one block of 32 x 32
// outputs as k_w8_tile<J, I> left it; a thread has 4 neighbouring ones, 8 threads a
// token's 32, so that loads and stores both go in pieces of 64 bytes or more.
template <int J, int I, int ACT>
__global__ __launch_bounds__(kBlock) void k_w8_join(W8Args a) {
  constexpr bool GATED = ACT != kNoAct;
  constexpr int IO = GATED ? I / 2 : I;
  int b = blockIdx.x;
  const int i = b % IO;
  b /= IO;
  const int j = b % J;
  b /= J;
  const int wave = b & 3, tile = b >> 2, tm = tile / a.tiles_n, tn = tile - tm * a.tiles_n;
  const int row = threadIdx.x >> 3, q = (threadIdx.x & 7) >> 1, h = threadIdx.x & 1;
  const int64_t m = static_cast<int64_t>(tm) * 64 * J + (wave & 1) * 32 * J + 32 * j + row;
  const int64_t n = static_cast<int64_t>(tn) * 64 * IO + (wave >> 1) * 32 * IO + 32 * i + 8 * q + 4 * h;
  if (m >= a.M || n >= a.N) return;
  const int64_t plane = static_cast<int64_t>(a.tiles_m) * a.tiles_n * (4 * J * I * 256);
  const i4v* src = reinterpret_cast<const i4v*>(a.part) +
                   (static_cast<int64_t>(tile) * 4 + wave) * (J * I * 256) + (j * I + i) * 256 + q * 64 + h * 32 + row;
  const float sx = a.sx[m * a.sx_step];
  f4v v[2];
#pragma unroll
  for (int p = 0; p < (GATED ? 2 : 1); ++p) {
    i4v s = {0, 0, 0, 0};
    for (int r = 0; r < a.splits; r += 4) {   // 4 loads under way at a time
      i4v v4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v4[e] = src[min(r + e, a.splits - 1) * plane + p * (I / 2 * 256)];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (r + e < a.splits) s += v4[e];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int64_t nc = n + c < a.N ? n + c : a.N - 1;
      v[p][c] = scaled(s[c], sx, a.sw[p][nc * a.sw_step[p]],
                       a.bias[p] ? ld_any(a.bias[p], a.bias_dt, nc) : 0.0f);
    }
  }
  if constexpr (GATED) {
#pragma unroll
    for (int c = 0; c < 4; ++c) v[0][c] = activate<ACT>(v[0][c]) * v[1][c];
  }
  st_quad(a, m, static_cast<int>(n), v[0]);
}

// K < 16 (0: the sums are empty): one output per thread, code by code.
template <int ACT>
__global__ __launch_bounds__(kBlock) void k_w8_short(W8Args a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
  if (i >= static_cast<int64_t>(a.M) * a.N) return;
  const int64_t m = i / a.N, n = i - m * a.N;
  const float sx = a.sx[m * a.sx_step];
  auto one = [&](int p) {
    int sum = 0;
    for (int k = 0; k < a.K; ++k)
      sum += static_cast<int8_t>(a.x[m * a.ldx + k]) * static_cast<int8_t>(a.w[p][n * a.ldw[p] + k]);
    return scaled(sum, sx, a.sw[p][n * a.sw_step[p]], a.bias[p] ? ld_any(a.bias[p], a.bias_dt, n) : 0.0f);
  };
  float v = one(0);
  if constexpr (ACT != kNoAct) v = activate<ACT>(v) * one(1);
  st_any(a.y, a.out_dt, i, v);
}

// Copies of x's rows and the weights' in rows of kp bytes (a multiple of 16), with
// zeros behind K: one launch for all, a thread per 16 bytes of the result.
struct W8Pad {
  const uint8_t* src[3];
  int64_t ld[3], first[4];   // first thread of each operand's copy, and the end
  uint8_t* dst;              // the copies, one behind the other
  int kp, K;
};

__global__ __launch_bounds__(kBlock) void k_w8_pad(W8Pad a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
  if (i >= a.first[3]) return;
  const int o = i >= a.first[2] ? 2 : i >= a.first[1] ? 1 : 0;
  const int cpr = a.kp >> 4;
  const int64_t c = i - (o == 2 ? a.first[2] : o ? a.first[1] : 0), r = c / cpr;
  const int k = static_cast<int>(c - r * cpr) * 16;
  const uint8_t* row = (o == 2 ? a.src[2] : o ? a.src[1] : a.src[0]) +
                       r * (o == 2 ? a.ld[2] : o ? a.ld[1] : a.ld[0]);
  *reinterpret_cast<u32x4*>(a.dst + i * 16) = from_k(ld_codes(row, k, a.K), k, a.K);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
size_t align256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

// The tiles: 256 x 256, 192 x 256 and 128 x 128, the last with four stages or, two
// workgroups per CU, with two.
enum { kT256, kT192, kT128, kT128x2, kTiles };
constexpr int kTileJ[] = {4, 3, 2, 2}, kTileI[] = {4, 4, 2, 2};

struct W8Plan {
  int few;                   // shape of cbq_w8a8_few.hip, or -1
  int tile, splits, split_steps;
  bool pad;                  // x and the weights are copied to rows of kp bytes first
  int64_t kp;
  size_t part_off, bytes;
};

// Modelled time in us of `tiles` tiles of steps_all k-steps, cut into sp ranges, for out
// sums (of both projections). A k-step takes longer the more CUs are busy (clock and
// bandwidth), a round adds the first loads and the outputs, ranges add a launch and
// their sums' traffic. Fitted to timings on MI355X (M = 130 .. 4096, N = 1024 .. 28672,
// K = 1024 .. 11008, one and two projections, 1 to 8 ranges of K): 9800 with aligned rows
// (7% off rms; what it picks is 0.8% slower on average than the best), 5700 each with
// rows of whole words and with others (8% and 7%; 1.6% and 1.5%).
struct W8Model { double step[kTiles], busy[kTiles], round[kTiles], two, call, join, sum; };
constexpr W8Model kModels[] = {
    {{1.13, 0.88, 0.35, 0.48}, {0.49, 0.39, 0.17, 0.215}, {7.4, 6.3, 3.3, 2.7}, 1.07, 3.0, 3.3, 1e-6},
    {{1.69, 0, 0, 0.62}, {0.51, 0, 0, 0.29}, {7.0, 0, 0, 2.6}, 1.46, 3.9, 3.0, 1e-6},
    {{2.12, 0, 0, 0.85}, {0.41, 0, 0, 0.40}, {6.9, 0, 0, 1.1}, 2.0, 6.3, 3.0, 0.86e-6}};

double w8_time(const W8Model& f, int tile, int64_t tiles, int64_t steps_all, int64_t out, int64_t sp, double cus) {
  const double wgs = static_cast<double>(tiles * sp), steps = static_cast<double>(cdiv(steps_all, sp));
  double t = f.call;
  auto once = [&](double n) { return steps * (f.step[tile] + f.busy[tile] * std::min(1.0, n / cus)) + f.round[tile]; };
  if (tile != kT128x2) {
    t += std::ceil(wgs / cus) * once(wgs);
  } else {   // two: a step of both workgroups of a CU
    const double full = std::floor(wgs / (2 * cus)), rem = wgs - full * 2 * cus;
    t += full * (steps * f.two + f.round[tile]);
    if (rem > cus) t += once(cus) + steps * (f.two - f.step[tile] - f.busy[tile]) * (rem - cus) / cus;
    else if (rem > 0) t += once(rem);
  }
  return sp > 1 ? t + f.join + f.sum * static_cast<double>(sp * out) : t;
}

constexpr int64_t kMaxTiles = 1 << 24;    // a grid has fewer than 2^32 threads, 256 to a tile

// room: bytes of workspace, or all that is wanted.
W8Plan w8_plan(int64_t M, int64_t N, int64_t K, int proj, int rows, size_t room = ~static_cast<size_t>(0)) {
  const int cus = device_cus();
  const int64_t steps = cdiv(K, 128);
  W8Plan p = {};
  p.bytes = CBQ_WS_CTRL_BYTES;
  const FewPlan few = M <= kFewRows ? few_plan(M, N, K, proj, rows, cus) : FewPlan{-1, 0.0};
  p.few = few.shape;
  // Mostly a third of the tiles' time, so the tiles' model is not asked; where they are close the
  // tiles may win (64 x 11008 x 4096, gated: 24 us, by tiles 22).
  if (M <= 64 && p.few >= 0) return p;
  p.kp = cdiv(K, 16) * 16;
  p.part_off = CBQ_WS_CTRL_BYTES;
  // Copies read and write M K + N K bytes at 4 TB/s and take a launch. Where rows are no
  // whole words the tiles win that back from about 640 tokens on, else hardly ever.
  const size_t copies = align256(static_cast<size_t>(M + proj * N) * p.kp);
  p.pad = rows == kRows1 && M >= 640 && p.part_off + copies <= room &&
          copies < (static_cast<size_t>(1) << 36);   // a grid has fewer than 2^32 threads
  if (p.pad) {
    p.part_off += copies;
    rows = kRows16;
  }
  double best = -1;
  p.splits = 1;
  for (int tile = 0; tile < kTiles; ++tile) {
    if (rows != kRows16 && (tile == kT192 || tile == kT128)) continue;
    const int64_t tiles = cdiv(M, 64 * kTileJ[tile]) * cdiv(N, 64 * kTileI[tile] / proj);
    if (tiles >= kMaxTiles) continue;
    const size_t plane = static_cast<size_t>(tiles) * kTileJ[tile] * kTileI[tile] * 16384;   // bytes of sums
    for (int64_t sp = 1; sp <= 8; ++sp) {
      const size_t bytes = p.part_off + (sp > 1 ? sp * plane : 0);
      if (sp > 1 && (tiles * sp > (tile == kT128x2 ? 2 : 1) * cus || steps / sp < 3 || bytes > room)) break;
      const double t = w8_time(kModels[rows], tile, tiles, steps, proj * M * N, sp, cus);
      if (best < 0 || t < best) {
        best = t;
        p.tile = tile;
        p.splits = static_cast<int>(sp);
        p.bytes = bytes;
      }
    }
  }
  if (p.few >= 0) {
    if (p.pad) best += 3.0 + static_cast<double>(copies) * 0.5e-6;
    if (few.us <= best) {
      p.pad = false;
      p.bytes = CBQ_WS_CTRL_BYTES;
      return p;
    }
    p.few = -1;
  }
  p.split_steps = static_cast<int>(cdiv(steps, p.splits));
  p.splits = static_cast<int>(cdiv(steps, p.split_steps));   // no empty ranges
  return p;
}

template <int J, int I, int NS, int ACT>
void launch_tile(const W8Args& a, bool any, hipStream_t s) {
  const unsigned tiles = static_cast<unsigned>(a.tiles_m) * a.tiles_n, grid = tiles * a.splits;
  constexpr int RAW = ACT == kNoAct ? kNoAct : CBQ_ACT_RELU;   // sums do not depend on it
  const bool split = a.splits > 1;
  if (any) {
    if constexpr (NS == 2 && J != 3) {
      if (split) k_w8_tile<J, I, 2, RAW, true, true><<<grid, 256, 0, s>>>(a);
      else k_w8_tile<J, I, 2, ACT, false, true><<<grid, 256, 0, s>>>(a);
    }
  } else if (split) {
    k_w8_tile<J, I, NS, RAW, true, false><<<grid, 256, 0, s>>>(a);
  } else {
    k_w8_tile<J, I, NS, ACT, false, false><<<grid, 256, 0, s>>>(a);
  }
  if (split) k_w8_join<J, I, ACT><<<tiles * 4 * J * (ACT == kNoAct ? I : I / 2), kBlock, 0, s>>>(a);
}

template <int ACT>
void launch_tiles(const W8Args& a, int tile, bool any, hipStream_t s) {
  switch (tile) {
    case kT256: launch_tile<4, 4, 2, ACT>(a, any, s); break;
    case kT192: launch_tile<3, 4, 2, ACT>(a, false, s); break;
    case kT128x2: launch_tile<2, 2, 2, ACT>(a, any, s); break;
    default: launch_tile<2, 2, 4, ACT>(a, false, s); break;
  }
}

constexpr int64_t kMaxStride = 1 << 22;   // 32-bit offsets within a tile's 256 rows

int check_rows(const char* what, const char* name, const cbq_i8_rows* r, int64_t rows, int64_t K) {
  CBQ_REQUIRE(r, "%s: %s is null", what, name);
  if (rows == 0) return CBQ_OK;
  CBQ_REQUIRE(r->scale && (K == 0 || r->data), "%s: %s has a null pointer", what, name);
  CBQ_REQUIRE(r->stride >= K && r->stride <= kMaxStride, "%s: %s rows are %lld bytes apart; expected %lld .. %lld",
              what, name, (long long)r->stride, (long long)K, (long long)kMaxStride);
  CBQ_REQUIRE(r->scale_stride == 0 || r->scale_stride == 1, "%s: %s scale_stride must be 0 or 1", what, name);
  return CBQ_OK;
}

// What rows of K codes are multiples of.
int rows_of(const cbq_i8_rows& r, int64_t K) {
  const uint64_t all = reinterpret_cast<uintptr_t>(r.data) | static_cast<uint64_t>(r.stride) | static_cast<uint64_t>(K);
  return all % 16 == 0 ? kRows16 : all % 4 == 0 ? kRows4 : kRows1;
}

int w8_run(const char* what, const cbq_i8_rows* x, const cbq_i8_rows* const (&w)[2], int proj,
           const void* const (&bias)[2], int bias_dtype, int act, int64_t M, int64_t N, int64_t K,
           void* y, int out_dtype, void* ws, size_t ws_bytes, cbq_stream_t stream) {
  clear_error();
  CBQ_REQUIRE(M >= 0 && N >= 0 && K >= 0, "%s: negative shape", what);
  CBQ_REQUIRE(M < (1LL << 31) - 256 && N < (1LL << 31) - 256, "%s: M and N must be below 2^31 - 256", what);
  CBQ_REQUIRE(K <= 131071, "%s: K must be at most 131071 (int32 sums), got %lld", what, (long long)K);
  CBQ_REQUIRE(out_dtype == CBQ_F32 || out_dtype == CBQ_F16 || out_dtype == CBQ_BF16,
              "%s: unsupported out_dtype %d", what, out_dtype);
  CBQ_REQUIRE((!bias[0] && !bias[1]) || bias_dtype == CBQ_F32 || bias_dtype == CBQ_F16 || bias_dtype == CBQ_BF16,
              "%s: unsupported bias dtype %d", what, bias_dtype);
  int rc = check_rows(what, "x", x, M, K);
  for (int p = 0; p < proj && rc == CBQ_OK; ++p)
    rc = check_rows(what, proj == 1 ? "w" : p ? "up" : "gate", w[p], N, K);
  if (rc != CBQ_OK) return rc;
  if (M == 0 || N == 0) return CBQ_OK;
  CBQ_REQUIRE(y, "%s: y is null", what);
  const int es = out_dtype == CBQ_F32 ? 4 : 2;
  CBQ_REQUIRE(aligned(y, es), "%s: y must be aligned to its elements", what);

  W8Args a = {};
  a.x = reinterpret_cast<const uint8_t*>(x->data);
  a.ldx = x->stride;
  a.sx = x->scale;
  a.sx_step = x->scale_stride;
  int rows = rows_of(*x, K);
  for (int p = 0; p < proj; ++p) {
    a.w[p] = reinterpret_cast<const uint8_t*>(w[p]->data);
    a.ldw[p] = w[p]->stride;
    a.sw[p] = w[p]->scale;
    a.sw_step[p] = w[p]->scale_stride;
    a.bias[p] = bias[p];
    rows = std::max(rows, rows_of(*w[p], K));
  }
  a.bias_dt = bias_dtype;
  a.act = act;
  a.y = y;
  a.out_dt = out_dtype;
  a.vec = N * es % 16 == 0 && aligned(y, 16);
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.splits = 1;
  hipStream_t s = as_stream(stream);
  if (K < 16) {
    CBQ_REQUIRE(M * N < (1LL << 32) - kBlock, "%s: fewer than 16 columns take less than 2^32 outputs", what);
    with_act(act, [&](auto c) {
      k_w8_short<decltype(c)::value><<<static_cast<unsigned>(cdiv(M * N, kBlock)), kBlock, 0, s>>>(a);
    });
    return launch_status(what);
  }
  const W8Plan p = w8_plan(M, N, K, proj, rows, ws && aligned(ws, 256) ? ws_bytes : 0);
  if (p.few >= 0) {
    launch_w8a8_few(a, p.few, rows != kRows16, s);
    return launch_status(what);
  }
  const int64_t tiles_m = cdiv(M, 64 * kTileJ[p.tile]), tiles_n = cdiv(N, 64 * kTileI[p.tile] / proj);
  CBQ_REQUIRE(tiles_m * tiles_n * p.splits < kMaxTiles, "%s: too many tiles", what);
  a.tiles_m = static_cast<int>(tiles_m);
  a.tiles_n = static_cast<int>(tiles_n);
  a.splits = p.splits;
  a.split_steps = p.split_steps;
  uint8_t* const w0 = static_cast<uint8_t*>(ws);
  if (p.pad) {
    W8Pad c = {{a.x, a.w[0], a.w[1]}, {a.ldx, a.ldw[0], a.ldw[1]}, {}, w0 + CBQ_WS_CTRL_BYTES,
               static_cast<int>(p.kp), a.K};
    const int64_t count[3] = {M, N, proj == 2 ? N : 0};
    for (int o = 0; o < 3; ++o) c.first[o + 1] = c.first[o] + count[o] * (p.kp / 16);
    const int64_t grid = cdiv(c.first[3], kBlock);
    k_w8_pad<<<static_cast<unsigned>(grid), kBlock, 0, s>>>(c);
    a.x = c.dst;
    a.w[0] = c.dst + c.first[1] * 16;
    a.w[1] = c.dst + c.first[2] * 16;
    a.ldx = a.ldw[0] = a.ldw[1] = p.kp;
    a.K = static_cast<int>(p.kp);   // zeros behind K
    rows = kRows16;
  }
  if (p.splits > 1) a.part = reinterpret_cast<int*>(w0 + p.part_off);
  with_act(act, [&](auto c) { launch_tiles<decltype(c)::value>(a, p.tile, rows != kRows16, s); });
  return launch_status(what);
}

}  // namespace
}  // namespace cbq

using namespace cbq;

extern "C" size_t cbq_w8a8_ws_bytes(int64_t M, int64_t N, int64_t K, int projections) {
  if (M <= 0 || N <= 0 || K < 16 || K > 131071 || projections < 1 || projections > 2)
    return CBQ_WS_CTRL_BYTES;
  return w8_plan(M, N, K, projections, K % 16 == 0 ? kRows16 : K % 4 == 0 ? kRows4 : kRows1).bytes;
}

extern "C" int cbq_w8a8_form_of(int64_t M, int64_t N, int64_t K, int projections, int multiple,
                                cbq_w8a8_form* form) {
  clear_error();
  const char* what = "cbq_w8a8_form_of";
  CBQ_REQUIRE(form, "%s: form is null", what);
  CBQ_REQUIRE(M > 0 && N > 0 && M < (1LL << 31) - 256 && N < (1LL << 31) - 256 && K >= 0 && K <= 131071,
              "%s: unsupported sizes", what);
  CBQ_REQUIRE(projections == 1 || projections == 2, "%s: projections must be 1 or 2, got %d", what, projections);
  CBQ_REQUIRE((multiple == 16 || multiple == 4 || multiple == 1) && K % multiple == 0,
              "%s: multiple must be 16, 4 or 1 and divide K, got %d", what, multiple);
  if (K < 16) {
    *form = {CBQ_W8A8_SHORT, 1, 1, kBlock, 0, 1, 0, cdiv(M * N, kBlock)};
    return CBQ_OK;
  }
  const int rows = multiple == 16 ? kRows16 : multiple == 4 ? kRows4 : kRows1;
  const W8Plan p = w8_plan(M, N, K, projections, rows);
  if (p.few >= 0) {
    *form = few_form(p.few, M, N, projections, rows);
    return CBQ_OK;
  }
  const int x_rows = 64 * kTileJ[p.tile], w_rows = 64 * kTileI[p.tile];
  *form = {CBQ_W8A8_TILES, w_rows, x_rows, 256, p.tile == kT128 ? 4 : 2, p.splits, p.pad,
           cdiv(M, x_rows) * cdiv(N, w_rows / projections) * p.splits};
  return CBQ_OK;
}

extern "C" int cbq_w8a8_linear(const cbq_i8_rows* x, const cbq_i8_rows* w, const void* bias,
                               int bias_dtype, int64_t M, int64_t N, int64_t K, void* y,
                               int out_dtype, void* ws, size_t ws_bytes, cbq_stream_t stream) {
  return w8_run("cbq_w8a8_linear", x, {w, nullptr}, 1, {bias, nullptr}, bias_dtype, kNoAct, M, N, K,
                y, out_dtype, ws, ws_bytes, stream);
}

extern "C" int cbq_w8a8_gated(const cbq_i8_rows* x, const cbq_i8_rows* gate, const cbq_i8_rows* up,
                              const void* gate_bias, const void* up_bias, int bias_dtype,
                              int activation, int64_t M, int64_t N, int64_t K, void* y,
                              int out_dtype, void* ws, size_t ws_bytes, cbq_stream_t stream) {
  clear_error();
  CBQ_REQUIRE(activation >= CBQ_ACT_SILU && activation <= CBQ_ACT_RELU,
              "cbq_w8a8_gated: unknown activation %d", activation);
  return w8_run("cbq_w8a8_gated", x, {gate, up}, 2, {gate_bias, up_bias}, bias_dtype, activation, M,
                N, K, y, out_dtype, ws, ws_bytes, stream);
}
