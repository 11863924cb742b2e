// cbq_kv.h - shared by the kernels of the 8-bit paged key/value cache: the
// batch as the kernels see it, the search for a workgroup's share of it, and
// the host's argument checks.
#pragma once

#include "cbq_device.h"
#include "cbq_host.h"
#include "cublade_kv.h"

namespace cbq {

enum : int { kKvInt8 = CBQ_KV_INT8, kKvFp8 = CBQ_KV_FP8 };

// Sequences of a call (by value in the kernels' arguments).
struct KvBatch {
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* cu;      // null: one new token per sequence
  int64_t tstride, tokens;
  int batch, max_pages;
  int page_shift;
  int num_pages;
};

// One sequence: its new tokens [tok0, tok0 + n) and its length with them. cu
// and lengths come from the device unchecked: the token range is cut to the
// call's tokens and the length to what the page table can hold.
struct KvSeq {
  int64_t tok0;
  int64_t n;
  int64_t len;
};

__device__ __forceinline__ KvSeq kv_seq(const KvBatch& m, int b) {
  KvSeq s;
  if (m.cu == nullptr) {
    s.tok0 = b;
    s.n = 1;
  } else {
    int64_t t0 = m.cu[b], t1 = m.cu[b + 1];
    t0 = t0 < 0 ? 0 : t0;
    t1 = t1 > m.tokens ? m.tokens : t1;
    s.tok0 = t0;
    s.n = t1 > t0 ? t1 - t0 : 0;
  }
  s.len = m.lengths[b];
  return s;
}

// Finds the sequence that owns work item `idx` when sequence b has count(seq)
// items and items are numbered sequence after sequence: returns b and sets rel to
// the item's number within it, or returns -1 past the last. Counts and their sum
// are below 2^31. All 64 lanes of a wave call it with the same idx: 64 sequences
// at a time, a scan over the lanes.
template <typename Count>
__device__ __forceinline__ int kv_find(const KvBatch& m, int idx, int& rel, Count count) {
  const int lane = threadIdx.x & 63;
  int run = 0;
  for (int b0 = 0; b0 < m.batch; b0 += 64) {
    int c = 0;
    if (b0 + lane < m.batch) c = count(kv_seq(m, b0 + lane));
    int incl = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(incl, o, 64);
      if (lane >= o) incl += up;
    }
    const uint64_t past = __ballot(run + incl > idx);
    if (past != 0) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(past)) - 1);
      rel = idx - run - __builtin_amdgcn_readlane(incl - c, l);
      return b0 + l;
    }
    run += __builtin_amdgcn_readlane(incl, 63);
  }
  return -1;
}

// Page id of page number p of sequence b, or -1 if it is not one of the pool.
__device__ __forceinline__ int kv_page(const KvBatch& m, int b, int64_t p) {
  if (p < 0 || p >= m.max_pages) return -1;
  const int id = m.table[b * m.tstride + p];
  return static_cast<uint32_t>(id) < static_cast<uint32_t>(m.num_pages) ? id : -1;
}

// Host side.
int kv_check_cache(const cbq_kv_cache* c);
int kv_check_batch(const cbq_kv_batch* b);
int kv_check_heads(const char* name, const cbq_kv_heads* h);
KvBatch kv_batch_of(const cbq_kv_cache* c, const cbq_kv_batch* b);

}  // namespace cbq
