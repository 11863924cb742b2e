// cbq_w8a8_few.hip - products of few rows of INT8 activations with INT8 weights
// (M <= 128): what counts is the stream of the weight, and then that of x.
//
//   y[m, n] = sx[m] sw[n] sum_k x[m, k] w[n, k] + bias[n]     or act(g) u of two
//
// k_w8_few<RT, MT, W, D, GATED, ANY>: a workgroup of W waves owns RT tiles of 16
// weight rows (gated: RT / 2 of the gate's and the same of the up projection's) and
// all MT tiles of 16 rows of x. Wave w takes the blocks w, w + W, ... of 128 bytes of
// k of all of them, so the waves share nothing until their sums meet. A unit (block,
// tile) is two loads of 8 rows x 128 bytes by LDS DMA: 8 lanes in a row fetch one
// cache line, while the matrix operand's own order (16 rows x 64 bytes, neighbouring
// lanes in different rows) takes the address unit 4 times as long. D blocks are in
// flight per wave in its own part of LDS, counted by vmcnt: no barrier, no registers.
// 16-byte chunk c of row r lies at c ^ (r & 7): no bank conflicts.
// v_mfma_i32_16x16x64_i8: A = weight rows, B = rows of x, so a lane ends with 4
// neighbouring outputs of one token.
//
// Bound: memory for 16 rows or less (N = 28672, K = 8192, M = 1: 39 us = 6.0 TB/s; M =
// 16, N = 11008, K = 4096: 9.9 us in a graph), then the reads of x by every workgroup.
// Measured against loads in the operand's order through registers (us, M = 16 / 32 /
// 64 / 128, N = K = 4096): 6.6 / 8.8 / 12.8 / 20.7 -> 5.8 / 5.9 / 7.3 / 11.3.
//
// Columns past K are zero in x, so that whatever the weight's load holds there does
// not count; rows past M and N repeat the last one and are not stored. ANY: rows that
// are no multiples of 16 bytes, which the DMA does not take: through registers, one
// block ahead.
#include <type_traits>

#include "cbq_lds_dma.h"
#include "cbq_w8a8.h"

namespace cbq {
namespace {

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <int RT, int MT, int W, int D, bool GATED, bool ANY>
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
  const int n0 = blockIdx.x * 16 * CT;
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
        off[u][h] = static_cast<uint32_t>(min((u - RT) * 16 + h * 8 + lrow, a.M - 1)) *
                    static_cast<uint32_t>(a.ldx);
      }
    }
  const uint8_t* base[3] = {a.w[0] + n0 * a.ldw[0], GATED ? a.w[1] + n0 * a.ldw[1] : nullptr, a.x};
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
    const int m = j * 16 + row, n = n0 + t * 16 + g * 4;
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

template <int RT, int MT, int W, int D, bool GATED>
void launch_few(const W8Args& a, hipStream_t s) {
  const int cols = 16 * (GATED ? RT / 2 : RT);
  const dim3 g(static_cast<unsigned>(cdiv(a.N, cols))), b(64 * W);
  const bool any = a.K % 16 || a.ldx % 16 || a.ldw[0] % 16 || !aligned(a.x, 16) || !aligned(a.w[0], 16) ||
                   (GATED && (a.ldw[1] % 16 || !aligned(a.w[1], 16)));
  if (any) k_w8_few<RT, MT, W, 1, GATED, true><<<g, b, 0, s>>>(a);
  else k_w8_few<RT, MT, W, D, GATED, false><<<g, b, 0, s>>>(a);
}

// Tiles per workgroup: the fewest that leave at most one workgroup per CU, with the
// most waves. Beyond that 4 tiles, so that fewer workgroups read x, and 4 waves, of
// which several fit a CU; but one tile where x is small beside the weight (us, RT = 1 /
// 4: N = 28672, K = 8192, M = 1 39 / 46, M = 16 45 / 46; N = 32000, K = 4096, M = 16
// 25 / 21; gated, RT = 2 / 4: N = 28672, K = 8192, M = 16 83 / 100, N = 14336, K = 4096
// 23 / 20).
template <int MT>
void launch_linear(const W8Args& a, hipStream_t s) {
  constexpr int W = MT == 8 ? 4 : 8;
  const int64_t cus = device_cus(), tiles = cdiv(a.N, 16);
  if (tiles <= cus) launch_few<1, MT, 8, MT == 1 ? 2 : 1, false>(a, s);
  else if (tiles <= 2 * cus) launch_few<2, MT, W, 1, false>(a, s);
  else if (tiles <= 3 * cus) launch_few<3, MT, W, 1, false>(a, s);
  else if (a.M <= 8 || (a.M <= 16 && tiles > 6 * cus)) launch_few<1, MT, 8, MT == 1 ? 2 : 1, false>(a, s);
  else launch_few<4, MT, 4, 1, false>(a, s);
}

template <int MT>
void launch_gated(const W8Args& a, hipStream_t s) {
  constexpr int W = MT == 8 ? 4 : 8;
  const int64_t cus = device_cus(), tiles = cdiv(a.N, 16);
  if (tiles <= cus || (a.M <= 32 && tiles > 6 * cus)) launch_few<2, MT, W, 1, true>(a, s);
  else if (tiles <= 2 * cus) launch_few<4, MT, W, 1, true>(a, s);
  else if (tiles <= 3 * cus) launch_few<6, MT, MT >= 4 ? 4 : 8, 1, true>(a, s);
  else launch_few<4, MT, 4, 1, true>(a, s);
}

}  // namespace

void launch_w8a8_few(const W8Args& a, hipStream_t s) {
  auto go = [&](auto mt) {
    constexpr int MT = decltype(mt)::value;
    if (a.act == kNoAct) launch_linear<MT>(a, s);
    else launch_gated<MT>(a, s);
  };
  if (a.M <= 16) go(std::integral_constant<int, 1>{});
  else if (a.M <= 32) go(std::integral_constant<int, 2>{});
  else if (a.M <= 64) go(std::integral_constant<int, 4>{});
  else go(std::integral_constant<int, 8>{});
}

}  // namespace cbq
