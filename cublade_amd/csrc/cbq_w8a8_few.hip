// cbq_w8a8_few.hip - products of few rows of INT8 activations with INT8
// weights (M <= 64): what counts is the stream of the weight.
//
//   y[m, n] = sx[m] sw[n] sum_k x[m, k] w[n, k] + bias[n]     or act(g) u of two
//
// k_w8_few<RT, MT, ACT, ANY>: an 8-wave workgroup owns RT tiles of 16 weight rows
// (gated: RT / 2 of the gate's and the same of the up projection's); wave w takes
// the blocks w, w + 8, ... of 128 bytes of k of all of them. A unit (block, tile)
// is two loads of 8 rows x 128 bytes straight from memory, which stream faster
// than the matrix operand's own 16 rows x 64 bytes; it goes through 2 KiB of the
// wave's own LDS into the operand's layout (16-byte chunk c of row r at c ^ (r &
// 7): no bank conflicts; a wave's LDS operations are in order, so compiler fences
// and no barrier). The activations come in the operand's layout straight from
// the L2 (every workgroup reads all M K of them). D blocks of loads are in flight
// per wave. v_mfma_i32_16x16x64_i8: A = weight rows, B = activation rows, so a
// lane ends with 4 neighbouring outputs of one token. The waves' sums meet in LDS
// (integers: any order gives the same).
//
// Columns past K are zero in x, so that whatever the weight's load holds there
// does not count; rows past M and N repeat the last one and are not stored.
#include <type_traits>

#include "cbq_lds_dma.h"
#include "cbq_w8a8.h"

namespace cbq {
namespace {

constexpr int kFewWaves = 8;
typedef u32x4 __attribute__((aligned(1))) u32x4_any;

// Blocks in flight per wave: 12 to 16 loads of the weight.
constexpr int few_depth(int rt) { return rt == 1 ? 6 : rt == 2 ? 4 : rt == 3 ? 2 : rt <= 6 ? 2 : 1; }

// 16 bytes at p + k of a row of K bytes, zero from K on. `k + 16 <= K` may not
// hold for a lane of the last block only.
template <bool ANY, bool NT>
__device__ __forceinline__ u32x4 ld_codes(const uint8_t* p, int k, int K) {
  if constexpr (!ANY) {
    const u32x4* q = reinterpret_cast<const u32x4*>(p + min(k, K - 16));
    const u32x4 v = NT ? __builtin_nontemporal_load(q) : *q;
    return k < K ? v : u32x4{0u, 0u, 0u, 0u};
  } else {
    if (k + 16 <= K) {
      const u32x4_any* q = reinterpret_cast<const u32x4_any*>(p + k);
      return NT ? __builtin_nontemporal_load(q) : *q;
    }
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    for (int j = 0; k + j < K; ++j) w[j >> 2] |= static_cast<uint32_t>(p[k + j]) << (8 * (j & 3));
    return u32x4{w[0], w[1], w[2], w[3]};
  }
}

template <int RT, int MT, int ACT, bool ANY>
__global__ __launch_bounds__(64 * kFewWaves) void k_w8_few(W8Args a) {
  constexpr bool GATED = ACT != kNoAct;
  constexpr int D = few_depth(RT);
  constexpr int CT = GATED ? RT / 2 : RT;           // tiles of 16 output columns
  static_assert(!GATED || RT % 2 == 0, "pairs of tiles");
  constexpr int kRed = RT * MT * kFewWaves * 1024;  // the waves' sums
  constexpr int kStage = kFewWaves * 2048;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kRed > kStage ? kRed : kStage];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16 * CT;
  uint8_t* const st = smem + wave * 2048;
  const int nblk = (a.K + 127) / 128;
  const int iters = (nblk + kFewWaves - 1) / kFewWaves;

  const uint8_t* wrow[RT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int p = GATED ? r & 1 : 0, t = GATED ? r >> 1 : r;
      wrow[r][h] = a.w[p] + min(n0 + t * 16 + h * 8 + (lane >> 3), a.N - 1) * a.ldw[p];
    }
  const uint8_t* xrow[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) xrow[j] = a.x + min(j * 16 + row, a.M - 1) * a.ldx;

  u32x4 w[D][RT][2], x[D][MT][2];
  auto load = [&](int i, int d) {
    const int b = i * kFewWaves + wave;
    if (b >= nblk) return;
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        x[d][j][e] = ld_codes<ANY, false>(xrow[j], b * 128 + e * 64 + g * 16, a.K);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[d][r][h] = ld_codes<ANY, true>(wrow[r][h], b * 128 + (lane & 7) * 16, a.K);
  };

  i4v acc[RT][MT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[r][j] = i4v{0, 0, 0, 0};

#pragma unroll
  for (int d = 0; d < D; ++d) load(d, d);
  const int wpos = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4);   // + 1024 for h = 1
  for (int i0 = 0; i0 < iters; i0 += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if ((i0 + d) * kFewWaves + wave < nblk) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          wave_lds_fence();   // the last unit is read before its stage is written
          *reinterpret_cast<u32x4*>(st + wpos) = w[d][r][0];
          *reinterpret_cast<u32x4*>(st + 1024 + wpos) = w[d][r][1];
          wave_lds_fence();   // written by all lanes before it is read
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const i4v fw = *reinterpret_cast<const i4v*>(st + row * 128 + (((g + 4 * e) ^ (row & 7)) << 4));
#pragma unroll
            for (int j = 0; j < MT; ++j)
              acc[r][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                  fw, __builtin_bit_cast(i4v, x[d][j][e]), acc[r][j], 0, 0, 0);
          }
        }
      }
      load(i0 + d + D, d);
    }
  }

  __syncthreads();   // every wave is past its stage
  i4v* red = reinterpret_cast<i4v*>(smem);
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int j = 0; j < MT; ++j) red[((r * MT + j) * kFewWaves + wave) * 64 + lane] = acc[r][j];
  __syncthreads();
  auto sum_of = [&](int r, int j) {
    const i4v* src = red + (r * MT + j) * kFewWaves * 64 + lane;
    i4v s = src[0];
#pragma unroll
    for (int v = 1; v < kFewWaves; ++v) s += src[v * 64];
    return s;
  };
  for (int q = wave; q < CT * MT; q += kFewWaves) {
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
      for (int c = 0; c < 4; ++c) v[0][c] = activate<ACT>(v[0][c]) * v[1][c];
    }
    st_quad(a, m, n, v[0]);
  }
}

template <int RT, int MT, int ACT>
void launch_few(const W8Args& a, hipStream_t s) {
  const int cols = 16 * (ACT == kNoAct ? RT : RT / 2);
  const dim3 g(static_cast<unsigned>(cdiv(a.N, cols))), b(64 * kFewWaves);
  const bool any = a.K % 16 || a.ldx % 16 || a.ldw[0] % 16 || !aligned(a.x, 16) || !aligned(a.w[0], 16) ||
                   (ACT != kNoAct && (a.ldw[1] % 16 || !aligned(a.w[1], 16)));
  if (any) k_w8_few<RT, MT, ACT, true><<<g, b, 0, s>>>(a);
  else k_w8_few<RT, MT, ACT, false><<<g, b, 0, s>>>(a);
}

template <int MT, int ACT>
void launch_few_mt(const W8Args& a, hipStream_t s) {
  // The fewest tiles that leave at most one workgroup per CU.
  const int64_t cus = device_cus();
  const int64_t tiles = cdiv(a.N, 16);
  if constexpr (ACT == kNoAct) {
    if (tiles <= cus) launch_few<1, MT, ACT>(a, s);
    else if (tiles <= 2 * cus || MT == 4) launch_few<2, MT, ACT>(a, s);
    else launch_few<3, MT, ACT>(a, s);
  } else {
    if (tiles <= cus || MT == 4) launch_few<2, MT, ACT>(a, s);
    else launch_few<4, MT, ACT>(a, s);
  }
}

}  // namespace

void launch_w8a8_few(const W8Args& a, hipStream_t s) {
  with_act(a.act, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    if (a.M <= 16) launch_few_mt<1, ACT>(a, s);
    else if (a.M <= 32) launch_few_mt<2, ACT>(a, s);
    else launch_few_mt<4, ACT>(a, s);
  });
}

}  // namespace cbq
