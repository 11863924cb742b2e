// cbq_w8a8.hip - products of INT8 activations and INT8 weights with a scale for
// each token and output channel, on gfx950 matrix cores, and the first half of a
// gated block: both projections, the activation and their product in one kernel.
//
//   y[m, n] = sx[m] sw[n] sum_k x[m, k] w[n, k] + bias[n]
//   y[m, n] = act(g) u,  g and u as above with the gate's and the up rows
//
// Sums are int32 and exact (K <= 131071). M <= 64: cbq_w8a8_few.hip.
//
// k_w8_tile<T, ACT, SPLIT>: T x T tiles (gated: T x T / 2 outputs, T / 2 columns of
// each projection side by side, so that a lane holds g and u of the same outputs) of
// v_mfma_i32_32x32x32_i8, 4 waves of T / 2 x T / 2. k-steps of 64 bytes; four LDS
// stages filled by LDS DMA, three k-steps in flight, one barrier per k-step between
// its two halves, so that the fragment reads of the next half overlap the products
// of this one.
//
// LDS layout of a stage: T rows of x, then T weight rows, 64 bytes each; 16-byte
// chunk c of row r at c ^ ((r >> 2) & 3). In half s of a k-step the lanes of half h
// (lane / 32) take chunk 2 h + s of both operands.
//
// A = weight rows, B = activation rows: lane l holds the outputs of token m = l % 32
// and n = 8 (v / 4) + 4 (l / 32) + v % 4. Outputs leave through LDS, 32 tokens at a
// time per wave, and are stored 16 bytes per lane along a row.
//
// K is cut into ranges where few tiles would leave CUs idle: each range writes its
// sums to the workspace and k_w8_join adds them (integers: exact in any order).
#include <type_traits>

#include "cbq_lds_dma.h"
#include "cbq_w8a8.h"

namespace cbq {
namespace {

constexpr int kW8NS = 4;   // LDS stages

template <int T> struct W8Geom {
  static constexpr int kWaves = 4;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kHalf = T * 64;                  // bytes of one operand per stage
  static constexpr int kSB = 2 * kHalf;
  static constexpr int kL = kHalf / (kThreads * 16);    // DMA instructions per operand
  static constexpr int kWT = T / 2;                     // edge of a wave's tile
  static constexpr int kJ = kWT / 32;                   // 32 x 32 tiles along its edges
  static constexpr int kPitch = kWT * 4 + 16;           // row of outputs in LDS, bytes
  static_assert(kWaves * 32 * kPitch <= kW8NS * kSB, "the outputs fit in the stages");
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

template <int T, int ACT, bool SPLIT>
__global__ __launch_bounds__(W8Geom<T>::kThreads) void k_w8_tile(W8Args a) {
  typedef W8Geom<T> G;
  constexpr bool GATED = ACT != kNoAct;
  constexpr int J = G::kJ, L = G::kL, WT = G::kWT, NW = G::kWaves;
  constexpr int TN = GATED ? T / 2 : T;                 // output columns of a tile
  constexpr int WN = GATED ? WT / 2 : WT;               // and of a wave
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kW8NS * G::kSB];
  __shared__ __attribute__((aligned(16))) float s_x[T], s_w[T], s_b[T];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int r32 = lane & 31, h = lane >> 5;
  const int tiles = a.tiles_m * a.tiles_n;
  const int split = SPLIT ? blockIdx.x / tiles : 0;
  int tm, tn;
  w8_tile(SPLIT ? blockIdx.x % tiles : blockIdx.x, a, tm, tn);
  const int m0 = tm * T, n0 = tn * TN;
  const int steps = a.K >> 6;                           // whole k-steps of all of K
  const int kb = split * a.split_steps;                 // first one of this range
  const int nk = SPLIT ? min(a.split_steps, steps - kb) : steps;
  const bool tail = (a.K & 63) && (!SPLIT || split == a.splits - 1);
  const uint32_t sbase = __builtin_amdgcn_readfirstlane(lds_addr(smem));

  // Weight row `r` of the tile: its projection, and its column from n0 on.
  // Gated: a wave's rows are WN of the gate, then the same WN of the up projection.
  auto proj_of = [&](int r) { return GATED ? (r % WT) / WN : 0; };
  auto col_of = [&](int r) { return GATED ? r / WT * WN + r % WN : r; };

  if constexpr (!SPLIT) {   // scales and biases of the tile's rows and columns
    for (int r = tid; r < T; r += G::kThreads) {
      s_x[r] = a.sx[min(m0 + r, a.M - 1) * a.sx_step];
      const int p = proj_of(r);
      const int64_t n = min(n0 + col_of(r), a.N - 1);
      s_w[r] = p ? a.sw[1][n * a.sw_step[1]] : a.sw[0][n * a.sw_step[0]];
      const void* b = p ? a.bias[1] : a.bias[0];
      s_b[r] = b ? ld_any(b, a.bias_dt, n) : 0.0f;
    }
  }

  // DMA instruction u of an operand fills rows (u NW + wave) 16 + lane / 4, chunk
  // slot lane % 4. Rows past M or N are the last row's; their products are not stored.
  const uint8_t* xbase = a.x + m0 * a.ldx;
  uint32_t xo[L], wo[L];
  const uint8_t* wbase[L];
#pragma unroll
  for (int u = 0; u < L; ++u) {
    const int row = (u * NW + wave) * 16 + (lane >> 2);
    const uint32_t c = static_cast<uint32_t>((lane & 3) ^ ((row >> 2) & 3)) << 4;
    const int p = __builtin_amdgcn_readfirstlane(proj_of(row));
    xo[u] = static_cast<uint32_t>(min(row, a.M - 1 - m0)) * static_cast<uint32_t>(a.ldx) + c;
    wo[u] = static_cast<uint32_t>(min(col_of(row), a.N - 1 - n0)) *
                static_cast<uint32_t>(p ? a.ldw[1] : a.ldw[0]) + c;
    wbase[u] = p ? a.w[1] + n0 * a.ldw[1] : a.w[0] + n0 * a.ldw[0];
  }
  auto issue_one = [&](int t, int stage, int u) {
    const uint32_t dst = sbase + stage * G::kSB + wave * 1024;
    if (u < L)
      lds_dma16(xo[u], uniform_ptr(xbase + static_cast<int64_t>(kb + t) * 64), dst + u * NW * 1024);
    else
      lds_dma16(wo[u - L], uniform_ptr(wbase[u - L] + static_cast<int64_t>(kb + t) * 64),
                dst + G::kHalf + (u - L) * NW * 1024);
  };

  uint32_t xr[2], wr[2];   // fragment read offsets of half s
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint32_t slot = static_cast<uint32_t>((2 * h + s) ^ ((r32 >> 2) & 3)) << 4;
    xr[s] = (wm * WT + r32) * 64 + slot;
    wr[s] = G::kHalf + (wn * WT + r32) * 64 + slot;
  }
  i16x acc[J][J];          // [token tile][weight tile]
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < J; ++i) acc[j][i] = i16x{};
  struct Frags { i4v x[J], w[J]; };
  auto read_one = [&](int stage, int s, Frags& f, int r) {
    const uint8_t* st = smem + stage * G::kSB;
    if (r < J) f.w[r] = *reinterpret_cast<const i4v*>(st + wr[s] + r * 2048);
    else f.x[r - J] = *reinterpret_cast<const i4v*>(st + xr[s] + (r - J) * 2048);
  };
  auto mma_one = [&](const Frags& f, int q) {
    acc[q / J][q % J] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[q % J], f.x[q / J],
                                                              acc[q / J][q % J], 0, 0, 0);
  };

  // Step t: f0 holds the fragments of tile t's first half. Its products run with the
  // reads of the second half into f1 between them; then the wait for tile t + 1 and
  // the barrier (every wave is past its reads of tile t - 1, whose stage tile t + 3
  // takes); then the second half's products, between them the DMA of tile t + 3 and
  // the reads of tile t + 1's first half.
  Frags f0, f1;
  auto step = [&](int t, auto dma, auto all) {
#pragma unroll
    for (int q = 0; q < J * J; ++q) {
      mma_one(f0, q);
#pragma unroll
      for (int r = 2 * J * q / (J * J); r < 2 * J * (q + 1) / (J * J); ++r)
        read_one(t % kW8NS, 1, f1, r);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (decltype(all)::value) dma_wait_barrier<0>();
    else dma_wait_barrier<2 * L>();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < J * J; ++q) {
      mma_one(f1, q);
#pragma unroll
      for (int r = 2 * J * q / (J * J); r < 2 * J * (q + 1) / (J * J); ++r)
        read_one((t + 1) % kW8NS, 0, f0, r);
      if constexpr (decltype(dma)::value) {
#pragma unroll
        for (int u = 2 * L * q / (J * J); u < 2 * L * (q + 1) / (J * J); ++u)
          issue_one(t + kW8NS - 1, (t + kW8NS - 1) % kW8NS, u);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using yes = std::true_type;
  using no = std::false_type;
#pragma unroll
  for (int t = 0; t < kW8NS - 1; ++t)
    if (t < nk) {
#pragma unroll
      for (int u = 0; u < 2 * L; ++u) issue_one(t, t, u);
    }
  if (nk > 0) {
    if (nk > 2) dma_wait_barrier<4 * L>();
    else if (nk > 1) dma_wait_barrier<2 * L>();
    else dma_wait_barrier<0>();
#pragma unroll
    for (int r = 0; r < 2 * J; ++r) read_one(0, 0, f0, r);
    int t = 0;
    for (; t + kW8NS - 1 < nk; ++t) step(t, yes{}, no{});
    if (t + 2 < nk) step(t++, no{}, no{});
    if (t + 1 < nk) step(t++, no{}, yes{});
#pragma unroll
    for (int r = 0; r < 2 * J; ++r) read_one((nk - 1) % kW8NS, 1, f1, r);
#pragma unroll
    for (int q = 0; q < J * J; ++q) mma_one(f0, q);
#pragma unroll
    for (int q = 0; q < J * J; ++q) mma_one(f1, q);
  }
  const int mw = m0 + wm * WT;
  if (tail) {   // the last K % 64 columns (a multiple of 16), straight from memory
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int k = steps * 64 + (2 * h + s) * 16;
      const bool in = k < a.K;
      const int kc = in ? k : 0;
#pragma unroll
      for (int i = 0; i < J; ++i) {
        const int r = wn * WT + 32 * i + r32, p = proj_of(wn * WT + 32 * i);
        const int64_t n = min(n0 + col_of(r), a.N - 1);
        f0.w[i] = *reinterpret_cast<const i4v*>((p ? a.w[1] : a.w[0]) +
                                                n * (p ? a.ldw[1] : a.ldw[0]) + kc);
        f0.x[i] = *reinterpret_cast<const i4v*>(a.x + min(mw + 32 * i + r32, a.M - 1) * a.ldx + kc);
        if (!in) f0.x[i] = i4v{0, 0, 0, 0};
      }
#pragma unroll
      for (int q = 0; q < J * J; ++q) mma_one(f0, q);
    }
  }

  // Outputs: 32 tokens at a time through the wave's own part of LDS.
  __syncthreads();
  uint8_t* const out = smem + wave * 32 * G::kPitch;
  const int nw = n0 + wn * WN;                          // the wave's first column
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int mj = mw + 32 * j;
    const float sx = SPLIT ? 0.0f : s_x[wm * WT + 32 * j + r32];
    wave_lds_fence();                                   // the last rows are read
#pragma unroll
    for (int i = 0; i < (GATED && !SPLIT ? J / 2 : J); ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = 32 * i + 8 * q + 4 * h;           // the wave's column of 4 outputs
        i4v bits;
        if constexpr (SPLIT) {
#pragma unroll
          for (int e = 0; e < 4; ++e) bits[e] = acc[j][i][4 * q + e];
        } else {
          const f4v w0 = *reinterpret_cast<const f4v*>(s_w + wn * WT + c);
          const f4v b0 = *reinterpret_cast<const f4v*>(s_b + wn * WT + c);
          f4v v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = scaled(acc[j][i][4 * q + e], sx, w0[e], b0[e]);
          if constexpr (GATED) {
            const f4v w1 = *reinterpret_cast<const f4v*>(s_w + wn * WT + WN + c);
            const f4v b1 = *reinterpret_cast<const f4v*>(s_b + wn * WT + WN + c);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = activate<ACT>(v[e]) * scaled(acc[j][i + J / 2][4 * q + e], sx, w1[e], b1[e]);
          }
          bits = __builtin_bit_cast(i4v, v);
        }
        *reinterpret_cast<i4v*>(out + r32 * G::kPitch + c * 4) = bits;
      }
    wave_lds_fence();                                   // written before it is read
    if constexpr (SPLIT) {
      // rows of T / 2 sums: gated, WN of each projection
#pragma unroll
      for (int r = 0; r < 32 * WT / 256; ++r) {
        const int e = (r * 64 + lane) * 4, row = e / WT, c = e % WT;
        const int p = GATED ? c / WN : 0;
        if (mj + row < a.M) {
          int* dst = a.part + ((static_cast<int64_t>(split) * (GATED ? 2 : 1) + p) * a.M + mj + row) * a.ldp;
          *reinterpret_cast<i4v*>(dst + nw + c % WN) =
              *reinterpret_cast<const i4v*>(out + row * G::kPitch + c * 4);
        }
      }
    } else if (a.vec && a.out_dt != kF32) {
#pragma unroll
      for (int r = 0; r < 32 * WN / 512; ++r) {
        const int e = (r * 64 + lane) * 8, row = e / WN, c = e % WN;
        const f4v lo = *reinterpret_cast<const f4v*>(out + row * G::kPitch + c * 4);
        const f4v hi = *reinterpret_cast<const f4v*>(out + row * G::kPitch + c * 4 + 16);
        const u32x4 o = a.out_dt == kF16
            ? u32x4{pack2_out<kF16>(lo.x, lo.y), pack2_out<kF16>(lo.z, lo.w),
                    pack2_out<kF16>(hi.x, hi.y), pack2_out<kF16>(hi.z, hi.w)}
            : u32x4{pack2_out<kBF16>(lo.x, lo.y), pack2_out<kBF16>(lo.z, lo.w),
                    pack2_out<kBF16>(hi.x, hi.y), pack2_out<kBF16>(hi.z, hi.w)};
        if (mj + row < a.M && nw + c < a.N)
          *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.y) +
                                    static_cast<int64_t>(mj + row) * a.N + nw + c) = o;
      }
    } else if (a.vec) {
#pragma unroll
      for (int r = 0; r < 32 * WN / 256; ++r) {
        const int e = (r * 64 + lane) * 4, row = e / WN, c = e % WN;
        const f4v v = *reinterpret_cast<const f4v*>(out + row * G::kPitch + c * 4);
        if (mj + row < a.M && nw + c < a.N)
          *reinterpret_cast<f4v*>(static_cast<float*>(a.y) + static_cast<int64_t>(mj + row) * a.N +
                                  nw + c) = v;
      }
    } else {
      for (int r = 0; r < 32 * WN / 64; ++r) {
        const int e = r * 64 + lane, row = e / WN, c = e % WN;
        const float v = *reinterpret_cast<const float*>(out + row * G::kPitch + c * 4);
        if (mj + row < a.M && nw + c < a.N)
          st_any(a.y, a.out_dt, static_cast<int64_t>(mj + row) * a.N + nw + c, v);
      }
    }
  }
}

// Adds the ranges' sums and finishes the outputs, four neighbouring ones per thread.
template <int ACT>
__global__ __launch_bounds__(kBlock) void k_w8_join(W8Args a) {
  constexpr int P = ACT != kNoAct ? 2 : 1;
  const int64_t quads = (a.N + 3) / 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
  if (i >= quads * a.M) return;
  const int64_t m = i / quads;
  const int n = static_cast<int>(i - m * quads) * 4;
  const float sx = a.sx[m * a.sx_step];
  f4v v[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int* src = a.part + (p * static_cast<int64_t>(a.M) + m) * a.ldp + n;
    i4v s = {0, 0, 0, 0};
    for (int r = 0; r < a.splits; ++r)
      s += *reinterpret_cast<const i4v*>(src + static_cast<int64_t>(r) * P * a.M * a.ldp);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int nc = min(n + c, a.N - 1);
      v[p][c] = scaled(s[c], sx, a.sw[p][nc * a.sw_step[p]],
                       a.bias[p] ? ld_any(a.bias[p], a.bias_dt, nc) : 0.0f);
    }
  }
  if constexpr (P == 2) {
#pragma unroll
    for (int c = 0; c < 4; ++c) v[0][c] = activate<ACT>(v[0][c]) * v[P - 1][c];
  }
  st_quad(a, m, n, v[0]);
}

// K = 0: the sums are empty.
template <int ACT>
__global__ __launch_bounds__(kBlock) void k_w8_empty(W8Args a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
  if (i >= static_cast<int64_t>(a.M) * a.N) return;
  const int64_t m = i / a.N, n = i - m * a.N;
  const float sx = a.sx[m * a.sx_step];
  auto one = [&](int p) {
    return scaled(0, sx, a.sw[p][n * a.sw_step[p]], a.bias[p] ? ld_any(a.bias[p], a.bias_dt, n) : 0.0f);
  };
  float v = one(0);
  if constexpr (ACT != kNoAct) v = activate<ACT>(v) * one(1);
  st_any(a.y, a.out_dt, i, v);
}

// Rows of K codes, ld bytes apart, as rows of kp bytes (a multiple of 64) with
// zeros behind them. One thread per 16 bytes of the result.
__global__ __launch_bounds__(kBlock) void k_w8_pad(const uint8_t* __restrict__ src, int64_t ld,
                                                   int64_t rows, int K, int64_t kp,
                                                   uint8_t* __restrict__ dst) {
  typedef u32x4 __attribute__((aligned(1))) u32x4_any;
  const int64_t cpr = kp >> 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
  if (i >= rows * cpr) return;
  const int64_t r = i / cpr;
  const int k = static_cast<int>(i - r * cpr) * 16;
  const uint8_t* p = src + r * ld + k;
  u32x4 v = {0u, 0u, 0u, 0u};
  if (k + 16 <= K) {
    v = *reinterpret_cast<const u32x4_any*>(p);
  } else {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    for (int j = 0; k + j < K; ++j) w[j >> 2] |= static_cast<uint32_t>(p[j]) << (8 * (j & 3));
    v = u32x4{w[0], w[1], w[2], w[3]};
  }
  *reinterpret_cast<u32x4*>(dst + i * 16) = v;
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
size_t align256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

struct W8Plan {
  int tile, splits, split_steps;
  int64_t ldp;               // columns of a plane of sums, a multiple of the tile's
  int64_t kp;                // K padded to whole steps
  size_t x_off, w_off[2], part_off, bytes;
};

// Tile and ranges of K: the pair with the lowest modelled time.
void w8_choose(int64_t M, int64_t N, int64_t nk, int proj, int& tile, int& splits) {
  const int64_t cus = device_cus();
  tile = 256;
  splits = 1;
  int64_t best = -1;
  for (int t : {256, 128}) {
    const int64_t tiles = cdiv(M, t) * cdiv(N, t / proj);
    const int64_t step = t == 256 ? 70 : 35;
    const int64_t max_wg = t == 256 ? cus : 2 * cus;
    for (int64_t sp = 1; sp <= 16; ++sp) {
      if (sp > 1 && (tiles * sp > max_wg || nk / sp < 4)) break;
      int64_t cost = step * cdiv(nk, sp) * cdiv(tiles * sp, cus);
      if (sp > 1) cost += 9 * cdiv(sp * M * N * proj * 4, 262144) + 400;
      if (best < 0 || cost < best) {
        best = cost;
        tile = t;
        splits = static_cast<int>(sp);
      }
    }
  }
}

// pad: x and the weights are copied to padded rows.
W8Plan w8_plan(int64_t M, int64_t N, int64_t K, int proj, bool pad) {
  W8Plan p;
  p.kp = cdiv(K, 64) * 64;
  size_t off = CBQ_WS_CTRL_BYTES;
  p.x_off = p.w_off[0] = p.w_off[1] = off;
  if (pad) {
    off = align256(off + static_cast<size_t>(M) * p.kp);
    for (int i = 0; i < proj; ++i) {
      p.w_off[i] = off;
      off = align256(off + static_cast<size_t>(N) * p.kp);
    }
  }
  const int64_t steps = pad ? p.kp / 64 : K / 64;
  w8_choose(M, N, steps, proj, p.tile, p.splits);
  p.split_steps = static_cast<int>(steps);
  if (p.splits > 1) {
    p.split_steps = static_cast<int>(cdiv(steps, p.splits));
    p.splits = static_cast<int>(cdiv(steps, p.split_steps));   // no empty ranges
  }
  p.ldp = cdiv(N, p.tile / proj) * (p.tile / proj);
  p.part_off = off;
  if (p.splits > 1) off = align256(off + static_cast<size_t>(p.splits) * proj * M * p.ldp * 4);
  p.bytes = off;
  return p;
}

template <int ACT>
void launch_tiles(const W8Args& a, int tile, hipStream_t s) {
  const unsigned tiles = static_cast<unsigned>(a.tiles_m) * a.tiles_n;
  constexpr int RAW = ACT == kNoAct ? kNoAct : CBQ_ACT_RELU;   // the sums do not depend on it
  if (a.splits > 1) {
    if (tile == 256) k_w8_tile<256, RAW, true><<<tiles * a.splits, W8Geom<256>::kThreads, 0, s>>>(a);
    else k_w8_tile<128, RAW, true><<<tiles * a.splits, W8Geom<128>::kThreads, 0, s>>>(a);
    const int64_t quads = static_cast<int64_t>(a.M) * ((a.N + 3) / 4);
    k_w8_join<ACT><<<static_cast<unsigned>(cdiv(quads, kBlock)), kBlock, 0, s>>>(a);
  } else if (tile == 256) {
    k_w8_tile<256, ACT, false><<<tiles, W8Geom<256>::kThreads, 0, s>>>(a);
  } else {
    k_w8_tile<128, ACT, false><<<tiles, W8Geom<128>::kThreads, 0, s>>>(a);
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

bool even16(const cbq_i8_rows& r) { return r.stride % 16 == 0 && aligned(r.data, 16); }

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
  bool pad = K % 16 || !even16(*x);
  for (int p = 0; p < proj; ++p) {
    a.w[p] = reinterpret_cast<const uint8_t*>(w[p]->data);
    a.ldw[p] = w[p]->stride;
    a.sw[p] = w[p]->scale;
    a.sw_step[p] = w[p]->scale_stride;
    a.bias[p] = bias[p];
    pad = pad || !even16(*w[p]);
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
  if (K == 0) {
    CBQ_REQUIRE(cdiv(M * N, kBlock) < (1LL << 31), "%s: too many outputs", what);
    with_act(act, [&](auto c) {
      k_w8_empty<decltype(c)::value><<<static_cast<unsigned>(cdiv(M * N, kBlock)), kBlock, 0, s>>>(a);
    });
    return launch_status(what);
  }
  if (M <= kFewRows) {
    launch_w8a8_few(a, s);
    return launch_status(what);
  }
  W8Plan p = w8_plan(M, N, K, proj, pad);
  const bool ws_ok = ws && aligned(ws, 256) && ws_bytes >= p.bytes;
  CBQ_REQUIRE(ws_ok || !pad, "%s: K, strides and addresses that are no multiples of 16 need a workspace of "
              "%zu bytes, 256-byte aligned", what, p.bytes);
  if (!ws_ok && p.splits > 1) {
    p.splits = 1;
    p.split_steps = static_cast<int>(K / 64);
  }
  a.tiles_m = static_cast<int>(cdiv(M, p.tile));
  a.tiles_n = static_cast<int>(cdiv(N, p.tile / proj));
  CBQ_REQUIRE(static_cast<int64_t>(a.tiles_m) * a.tiles_n * p.splits < (1LL << 31) &&
                  cdiv(M * cdiv(N, 4), kBlock) < (1LL << 31), "%s: too many tiles", what);
  a.splits = p.splits;
  a.split_steps = p.split_steps;
  uint8_t* base = static_cast<uint8_t*>(ws);
  if (pad) {
    auto copy = [&](const uint8_t*& src, int64_t& ld, int64_t rows, size_t off) {
      const int64_t n = rows * (p.kp / 16);
      k_w8_pad<<<static_cast<unsigned>(cdiv(n, kBlock)), kBlock, 0, s>>>(src, ld, rows, a.K, p.kp, base + off);
      src = base + off;
      ld = p.kp;
    };
    CBQ_REQUIRE(cdiv((M > N ? M : N) * (p.kp / 16), kBlock) < (1LL << 31), "%s: too many rows", what);
    copy(a.x, a.ldx, M, p.x_off);
    for (int i = 0; i < proj; ++i) copy(a.w[i], a.ldw[i], N, p.w_off[i]);
    a.K = static_cast<int>(p.kp);
  }
  a.part = reinterpret_cast<int*>(base + p.part_off);
  a.ldp = p.ldp;
  with_act(act, [&](auto c) { launch_tiles<decltype(c)::value>(a, p.tile, s); });
  return launch_status(what);
}

}  // namespace
}  // namespace cbq

using namespace cbq;

extern "C" size_t cbq_w8a8_ws_bytes(int64_t M, int64_t N, int64_t K, int projections) {
  if (M <= kFewRows || N <= 0 || K <= 0 || K > 131071 || projections < 1 || projections > 2)
    return CBQ_WS_CTRL_BYTES;
  return w8_plan(M, N, K, projections, K % 16 != 0).bytes;
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
