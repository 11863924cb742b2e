// cbq_w8a8_few.hip - products of few rows of INT8 activations with INT8 weights, and
// small products: too few outputs for the tiles of cbq_w8a8.hip to fill the chip.
//
//   y[m, n] = sx[m] sw[n] sum_k x[m, k] w[n, k] + bias[n]     or act(g) u of two
//
// k_w8_few<RT, MT, W, D, GATED, ANY, ONE>: a workgroup of W waves owns RT tiles of 16
// weight rows (gated: RT / 2 of the gate's and the same of the up projection's) and
// MT tiles of 16 rows of x. Wave w takes the blocks w, w + W, ... of 128 bytes of
// k of all of them, so the waves share nothing until their sums meet. A unit (block,
// tile) is two loads of 8 rows x 128 bytes by LDS DMA: 8 lanes in a row fetch one
// cache line, while the matrix operand's own order (16 rows x 64 bytes, neighbouring
// lanes in different rows) takes the address unit 4 times as long. D blocks are in
// flight per wave in its own part of LDS, counted by vmcnt: no barrier, no registers.
// 16-byte chunk c of row r lies at c ^ (r & 7): no bank conflicts.
// v_mfma_i32_16x16x64_i8: A = weight rows, B = rows of x, so a lane ends with 4
// neighbouring outputs of one token.
//
// Bound: memory for 16 rows or less (N = 28672, K = 8192, M = 1: 45 us = 5.3 TB/s; M =
// 16, N = 11008, K = 4096: 9.7 us), then the reads of x by every workgroup, and for small
// products the chain of loads, sums and stores. Blocks of 16 or 32 rows of x, each with
// workgroups of its own, beat workgroups with all rows there, since more waves load (us,
// M = 64 / 128, N = K = 4096: 7.3 / 11.3 -> 6.8 / 8.2), and beat the tiles, whose 256
// threads own 128 x 128 outputs or more (M = 333, N = 1001, K = 1403: 12 -> 7.4; M = 256,
// N = K = 4096: 17 -> 11).
// Measured against loads in the operand's order through registers (us, M = 16 / 32 /
// 64 / 128, N = K = 4096): 6.6 / 8.8 / 12.8 / 20.7 -> 5.8 / 5.9 / 7.3 / 11.3.
//
// Columns past K are zero in x, so that whatever the weight's load holds there does
// not count; rows past M and N repeat the last one and are not stored. ANY: rows that
// are no multiples of 16 bytes, which the DMA does not take: through registers, one
// block ahead.
#include <algorithm>
#include <type_traits>

#include "cbq_lds_dma.h"
#include "cbq_w8a8.h"

namespace cbq {
namespace {

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <int RT, int MT, int W, int D, bool GATED, bool ANY, bool ONE>
__global__ __launch_bounds__(64 * W) void k_w8_few(W8Args a) {
  constexpr int CT = GATED ? RT / 2 : RT;           // tiles of 16 output columns
  static_assert(!GATED || RT % 2 == 0, "pairs of tiles");
  constexpr int U = RT + MT;                        // units of a block: 16 rows x 128 bytes
  constexpr int NOPS = 2 * U;                       // loads of a block
  static_assert(NOPS * D <= 63, "loads in flight are counted in 6 bits");
  __shared__ __attribute__((aligned(1024))) uint8_t ring[W * D * U * 2048];
  __shared__ __attribute__((aligned(16))) int red[RT * MT * 256];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = lane & 15, g = lane >> 4;
  // Workgroups of the same weight rows run on one XCD (b % 8), one after the other, so
  // that its L2 reads them once (M = 64, N = 11008, K = 4096, 16 rows of x each: 23 us
  // -> 16). The grid is a whole number of rounds over the XCDs. ONE: one block of rows of
  // x and no such order, which would cost single tokens 0.3 us.
  int n0 = blockIdx.x, m0 = 0;
  if constexpr (!ONE) {
    const int turn = n0 >> 3;
    m0 = turn % a.tiles_m * 16 * MT;
    n0 = turn / a.tiles_m * 8 + (n0 & 7);
    if (n0 * 16 * CT >= a.N) return;
  }
  n0 *= 16 * CT;
  uint8_t* const mine = ring + wave * (D * U * 2048);
  const uint32_t mine_lds = __builtin_amdgcn_readfirstlane(lds_addr(mine));
  const int nblk = (a.K + 127) / 128;
  const int iters = (nblk - wave + W - 1) / W;      // blocks of this wave
  for (int i = tid; i < RT * MT * 256; i += 64 * W) red[i] = 0;

  // Load h of a unit: rows 8 h + lane / 8, the chunk that belongs at slot lane % 8.
  const int lrow = lane >> 3;
  const int lk = ((lane & 7) ^ lrow) << 4;          // byte of the chunk in its block (row & 7 = lrow)
  uint32_t off[U][2];                               // of the row, from the unit's base
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (u < RT) {
        const int p = GATED ? u & 1 : 0, t = GATED ? u >> 1 : u;
        off[u][h] = static_cast<uint32_t>(min(t * 16 + h * 8 + lrow, a.N - 1 - n0)) *
                    static_cast<uint32_t>(a.ldw[p]);
      } else {
        off[u][h] = static_cast<uint32_t>(min((u - RT) * 16 + h * 8 + lrow, a.M - 1 - m0)) *
                    static_cast<uint32_t>(a.ldx);
      }
    }
  const uint8_t* base[3] = {a.w[0] + n0 * a.ldw[0], GATED ? a.w[1] + n0 * a.ldw[1] : nullptr, a.x + m0 * a.ldx};
  auto base_of = [&](int u) { return u >= RT ? base[2] : GATED && (u & 1) ? base[1] : base[0]; };
  u32x4 held[ANY ? U : 1][2];                       // ANY: loads on their way to LDS
  auto fetch = [&](int i, int slot) {
    const int k = min((i * W + wave) * 128 + lk, a.K - 16);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (ANY) held[u][h] = ld_codes(base_of(u) + off[u][h], (i * W + wave) * 128 + lk, a.K);
        else
          lds_dma16(off[u][h] + static_cast<uint32_t>(k), uniform_ptr(base_of(u)),
                    mine_lds + (slot * U + u) * 2048 + h * 1024);
      }
  };

  i4v acc[RT][MT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[r][j] = i4v{0, 0, 0, 0};

  constexpr int DD = ANY ? 1 : D;
#pragma unroll
  for (int d = 0; d < DD; ++d)
    if (d < iters) fetch(d, d);
  auto block = [&](int i, int slot) {
    const int b = i * W + wave;
    uint8_t* st = mine + slot * U * 2048;
    if constexpr (ANY) {
      wave_lds_fence();   // the last block is read before its stage is written
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<u32x4*>(st + u * 2048 + h * 1024 + lane * 16) =
              from_k(held[u][h], b * 128 + lk, a.K);
      wave_lds_fence();   // written by all lanes before it is read
      if (i + 1 < iters) fetch(i + 1, 0);
    }
    i4v f[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        f[u][e] = *reinterpret_cast<const i4v*>(st + u * 2048 + row * 128 + (((g + 4 * e) ^ (row & 7)) << 4));
    if constexpr (!ANY) {
      if (b == nblk - 1 && (a.K & 127)) {   // chunks of x behind K count as zeros
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (b * 128 + (g + 4 * e) * 16 >= a.K) f[RT + j][e] = i4v{0, 0, 0, 0};
      }
      if (i + D < iters) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the stage is read
        fetch(i + D, slot);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int j = 0; j < MT; ++j)
          acc[r][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[r][e], f[RT + j][e], acc[r][j], 0, 0, 0);
  };
  if constexpr (ANY) {
    for (int i = 0; i < iters; ++i) block(i, 0);
  } else {
    int i = 0;
    for (; i + 2 * D <= iters; i += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        wait_vm<(D - 1) * NOPS>();
        block(i + d, d);
      }
    }
    for (; i < iters; ++i) {   // fewer than D blocks may follow
      wait_vm<0>();
      block(i, i % D);
    }
  }
  // The waves' sums meet in LDS: integers, so their order does not matter.
  __syncthreads();   // the sums are zero
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) atomicAdd(red + (r * MT + j) * 256 + c * 64 + lane, acc[r][j][c]);
  __syncthreads();
  auto sum_of = [&](int r, int j) {
    const int* src = red + (r * MT + j) * 256 + lane;
    return i4v{src[0], src[64], src[128], src[192]};
  };
  for (int q = wave; q < CT * MT; q += W) {
    const int t = q / MT, j = q % MT;
    const int m = m0 + j * 16 + row, n = n0 + t * 16 + g * 4;
    if (m >= a.M || n >= a.N) continue;
    const float sx = a.sx[m * a.sx_step];
    f4v v[2];
#pragma unroll
    for (int p = 0; p < (GATED ? 2 : 1); ++p) {
      const i4v s = sum_of(GATED ? 2 * t + p : t, j);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int nc = min(n + c, a.N - 1);
        v[p][c] = scaled(s[c], sx, a.sw[p][nc * a.sw_step[p]],
                         a.bias[p] ? ld_any(a.bias[p], a.bias_dt, nc) : 0.0f);
      }
    }
    if constexpr (GATED) {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[0][c] = activate(a.act, v[0][c]) * v[1][c];
    }
    st_quad(a, m, n, v[0]);
  }
}

// The shapes a workgroup comes in (6 tiles of weight rows: gated only).
struct FewShape { int rt, mt, waves, depth; };
constexpr FewShape kShapes[] = {{1, 1, 8, 2}, {2, 1, 8, 1}, {3, 1, 8, 1}, {4, 1, 4, 1}, {6, 1, 8, 1},
                                {1, 2, 8, 1}, {2, 2, 8, 1}, {3, 2, 8, 1}, {4, 2, 4, 1},
                                {2, 4, 8, 1}, {3, 4, 8, 1}, {4, 4, 4, 1}, {4, 4, 8, 1}};
constexpr int kNumShapes = sizeof(kShapes) / sizeof(kShapes[0]);

// Modelled time in us of a shape: a call, a round of as many workgroups as fit the CUs
// (counted on the fullest XCD), a wave's blocks in it (step; more for each further
// workgroup of the CU), and the weights' megabytes (far: those past 90). Fitted to
// timings on MI355X (M = 1 .. 1024, N = 200 .. 32000, K = 200 .. 14336, one and two
// projections): 2400 with aligned rows, 1200 each with rows of whole words and with
// others. A time is 10% off rms; what the model picks is 1% slower on average than the
// fastest of the shapes.
struct FewModel { double call, round, step, more, mb, far; };
constexpr FewModel kFewModels[][kNumShapes] = {
    {{1.65, 0.819, 0.216, 0.258, 0.0832, 0.0742}, {1.89, 0.778, 0.316, 0.352, 0.105, 0.0611},
     {1.88, 0.749, 0.417, 0.541, 0.0982, 0.0825}, {1.43, 1.45, 0.399, 0.229, 0.103, 0.0713},
     {1.19, 1.87, 0.934, 0, 0.0995, 0.0668}, {2.09, 0.578, 0.381, 0.47, 0.0586, 0.113},
     {1.8, 1.19, 0.515, 0.626, 0.0746, 0.0801}, {1.34, 1.47, 0.704, 0, 0.0696, 0.129},
     {1.5, 2.01, 0.539, 0.319, 0.0821, 0.0991}, {1.37, 1.83, 0.861, 0, 0.0677, 0.121},
     {1.23, 2.42, 1.01, 0, 0.072, 0.113}, {1.35, 3.95, 0.671, 0.487, 0.0812, 0.0862},
     {1.34, 2.62, 1.16, 0, 0.0876, 0.0897}},
    {{2.17, 0.422, 0.299, 0.377, 0.0786, 0.141}, {2.08, 0.778, 0.448, 0.563, 0.101, 0.0812},
     {1.72, 1.13, 0.587, 0.711, 0.106, 0.101}, {2.3, 0.995, 0.51, 0.536, 0.0936, 0.0888},
     {1.19, 2.01, 1.48, 0, 0.114, 0.0646}, {2.2, 0.501, 0.576, 0.587, 0.0722, 0.244},
     {1.81, 1.23, 0.802, 0.724, 0.0813, 0.128}, {1.27, 1.85, 0.996, 0, 0.0976, 0.182},
     {1.76, 2.2, 0.691, 0.553, 0.0888, 0.113}, {1.27, 2.19, 1.23, 0, 0.0897, 0.14},
     {1.18, 2.86, 1.46, 0, 0.101, 0.18}, {1.59, 4.31, 0.995, 0.809, 0.0763, 0.119},
     {1.22, 3.08, 1.77, 0, 0.105, 0.0888}},
    {{2.37, 0, 0.709, 0.661, 0.0326, 0.146}, {2.11, 0.498, 1.02, 0.9, 0.0594, 0.111},
     {1.77, 0.663, 1.36, 1.17, 0.0619, 0.116}, {2.56, 0.687, 0.851, 0.892, 0.0604, 0.093},
     {0.99, 1.7, 2.56, 0, 0.0713, 0.0769}, {2.4, 0, 1.11, 0.819, 0.0905, 0.188},
     {2.28, 0.482, 1.4, 1.17, 0.0789, 0.107}, {1.55, 1.25, 1.74, 0, 0.0721, 0.15},
     {2.15, 1.74, 1.05, 0.967, 0.0666, 0.104}, {1.53, 1.54, 2.09, 0, 0.0851, 0.131},
     {1.42, 2.12, 2.47, 0, 0.0761, 0.131}, {1.93, 3.94, 1.47, 1.29, 0.0614, 0.123},
     {1.55, 2.35, 2.8, 0, 0.0893, 0.0819}}};

template <int RT, int MT, int W, int D, bool GATED>
void launch_few(W8Args a, bool any, hipStream_t s) {
  const unsigned blocks_n = static_cast<unsigned>(cdiv(a.N, 16 * (GATED ? RT / 2 : RT)));
  if constexpr (MT == 1) {
    if (a.M <= 16) {
      if (any) k_w8_few<RT, 1, W, 1, GATED, true, true><<<blocks_n, 64 * W, 0, s>>>(a);
      else k_w8_few<RT, 1, W, D, GATED, false, true><<<blocks_n, 64 * W, 0, s>>>(a);
      return;
    }
  }
  a.tiles_m = static_cast<int>(cdiv(a.M, 16 * MT));
  const unsigned g = static_cast<unsigned>(cdiv(blocks_n, 8)) * 8 * a.tiles_m;
  if (any) k_w8_few<RT, MT, W, 1, GATED, true, false><<<g, 64 * W, 0, s>>>(a);
  else k_w8_few<RT, MT, W, D, GATED, false, false><<<g, 64 * W, 0, s>>>(a);
}

}  // namespace

cbq_w8a8_form few_form(int shape, int64_t M, int64_t N, int proj, int rows) {
  const FewShape& f = kShapes[shape];
  cbq_w8a8_form r = {CBQ_W8A8_FEW, 16 * f.rt, 16 * f.mt, 64 * f.waves, rows == kRows16 ? f.depth : 1, 1, 0, 0};
  r.workgroups = cdiv(N, 16 * (f.rt / proj));
  if (f.mt > 1 || M > 16) r.workgroups = cdiv(r.workgroups, 8) * 8 * cdiv(M, r.x_rows);   // see launch_few
  return r;
}

FewPlan few_plan(int64_t M, int64_t N, int64_t K, int proj, int rows, int cus) {
  FewPlan best = {-1, 0.0};
  for (int c = 0; c < kNumShapes; ++c) {
    const FewShape& f = kShapes[c];
    // Tiles of x that hold no rows cost what others do, and many blocks of 16 rows of x
    // read the weight as often.
    if (f.rt % proj || (f.rt == 6 && proj == 1) || (f.mt > 1 && M <= 8 * f.mt) || (f.mt == 1 && M > 64)) continue;
    const int64_t wgs = cdiv(cdiv(N, 16 * (f.rt / proj)), 8) * 8 * cdiv(M, 16 * f.mt), steps = cdiv(cdiv(K, 128), f.waves);
    if (wgs * f.waves >= 1 << 26) continue;   // a grid has fewer than 2^32 threads
    const int64_t lds = f.waves * (rows == kRows16 ? f.depth : 1) * (f.rt + f.mt) * 2048 + f.rt * f.mt * 1024;
    const int64_t per_cu = std::min<int64_t>(160 * 1024 / lds, 2048 / (64 * f.waves));
    const int64_t full = wgs / (per_cu * cus), rem = wgs - full * per_cu * cus;
    const int64_t rounds = full + (rem > 0), more = full * (per_cu - 1) + (rem > 0 ? cdiv(rem, cus) - 1 : 0);
    const FewModel& m = kFewModels[rows][c];
    const double mb = 1e-6 * static_cast<double>(proj * N * K);
    const double us = m.call + rounds * m.round + static_cast<double>(steps) * (rounds * m.step + more * m.more) +
                      mb * m.mb + std::max(0.0, mb - 90) * m.far;
    if (best.shape < 0 || us < best.us) best = {c, us};
  }
  return best;
}

void launch_w8a8_few(const W8Args& a, int shape, bool any, hipStream_t s) {
  auto go = [&](auto c) {
    constexpr FewShape F = kShapes[decltype(c)::value];
    if constexpr (F.rt % 2 == 0) {
      if (a.act != kNoAct) return launch_few<F.rt, F.mt, F.waves, F.depth, true>(a, any, s);
    }
    if constexpr (F.rt < 6) launch_few<F.rt, F.mt, F.waves, F.depth, false>(a, any, s);
  };
  auto pick = [&](auto&& self, auto c) {
    if (shape == decltype(c)::value) go(c);
    else if constexpr (decltype(c)::value + 1 < kNumShapes)
      self(self, std::integral_constant<int, decltype(c)::value + 1>{});
  };
  pick(pick, std::integral_constant<int, 0>{});
}

}  // namespace cbq
