// Shared pieces of the long-context kernels: sequences over a paged cache, and the choice of the
// largest values of a row.
#pragma once

#include <stdint.h>

#include "ifa4_internal.h"
#include "ifa4_ptx.cuh"

namespace ifa4 {

// Sequence of row t: cu_q[b] <= t < cu_q[b + 1], -1 for a row of none.  Whole warp; 32 places are
// looked at a time (one step for up to 33 sequences, two for 1057).
__device__ __forceinline__ int find_sequence(const int32_t* cu_q, int batch, long long t) {
  const int lane = threadIdx.x & 31;
  // one sequence a row is the usual decode batch
  const int guess = t < batch ? static_cast<int>(t) : batch - 1;
  const int32_t ends = __ldg(cu_q + (lane == 0 ? 0 : lane == 1 ? batch : guess + (lane & 1)));
  if (t < __shfl_sync(0xffffffffu, ends, 0) || t >= __shfl_sync(0xffffffffu, ends, 1)) return -1;
  if (__shfl_sync(0xffffffffu, ends, 2) <= t && t < __shfl_sync(0xffffffffu, ends, 3)) return guess;
  int lo = 0, hi = batch;  // cu_q[lo] <= t < cu_q[hi]
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = min(lo + (lane + 1) * step, hi);
    const unsigned le = __ballot_sync(0xffffffffu, at < hi && __ldg(cu_q + at) <= t);
    const int n = __popc(le);  // offsets ascend: the first n places
    hi = min(lo + (n + 1) * step, hi);
    lo += n * step;
  }
  return lo;
}

// Page of entry c of a table row, -1 for none.
__device__ __forceinline__ int page_at(const PagedSeqs& s, const int32_t* table_row, int c) {
  if (c < 0 || c >= s.table_width) return -1;
  const int p = __ldg(table_row + c);
  return p >= 0 && p < s.num_pages ? p : -1;
}
__device__ __forceinline__ const int32_t* table_row(const PagedSeqs& s, int b) {
  return s.block_table + static_cast<long long>(b) * s.bt_stride;
}

// ---------------------------------------------------------------------------------------
// The `count` largest of a row
// ---------------------------------------------------------------------------------------
// Order-preserving image of a float: -inf is 0 (never chosen), NaN is above +inf, the zeros are
// equal; kAlways is above all of them.
constexpr uint32_t kAlways = 0xffffffffu;
__device__ __forceinline__ uint32_t rank_of(float x) {
  const uint32_t b = __float_as_uint(x);
  if ((b & 0x7fffffffu) > 0x7f800000u) return kAlways - 1u;
  if (b == 0xff800000u) return 0u;
  if ((b & 0x7fffffffu) == 0u) return 0x80000000u;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

template <int kThreads>
struct SelectSmem {
  uint32_t hist[2048];
  uint32_t warp[kThreads / 32];
  uint32_t digit, above, total, in_bin;
};

// Exclusive sum over the threads of a block, and the total; two barriers.
template <int kThreads>
__device__ __forceinline__ uint32_t block_exclusive_sum(uint32_t v, uint32_t* warp_sums,
                                                        uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += up;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  constexpr int kWarps = kThreads / 32;
  const uint32_t w = lane < kWarps ? warp_sums[lane] : 0u;
  uint32_t winc = w;
#pragma unroll
  for (int d = 1; d < kWarps; d <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, winc, d);
    if (lane >= d) winc += up;
  }
  total = __shfl_sync(0xffffffffu, winc, kWarps - 1);
  const uint32_t before = __shfl_sync(0xffffffffu, winc - w, warp);
  __syncthreads();
  return before + inc - v;
}

// Calls emit(place, i) for the `count` elements of the largest key(i), 0 <= i < n, in ascending i;
// elements of key 0 are never taken, of equal ones at the border the lowest i are.  Whole block.
// Returns how many there are.  Three passes over digits of 11, 11 and 10 bits find the key of the
// border, one more writes what is above it; each reads the row again, which the caches hold.
template <int kThreads, class Key, class Emit>
__device__ __forceinline__ int select_largest(SelectSmem<kThreads>& sm, int n, int count, Key key,
                                              Emit emit) {
  const int tid = threadIdx.x;
  uint32_t need = static_cast<uint32_t>(count), prefix = 0u, known = 0u;
  bool all = false, bin_whole = false;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const int bins = pass == 2 ? 1024 : 2048;
    for (int i = tid; i < bins; i += kThreads) sm.hist[i] = 0u;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const uint32_t u = key(i);
      if (u != 0u && (u & known) == prefix) atomicAdd(&sm.hist[(u >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    // thread 0 has the highest bins
    const int per = bins / kThreads > 0 ? bins / kThreads : 1;
    const int top = bins - 1 - tid * per;
    uint32_t mine = 0u;
    if (top >= 0)
      for (int j = 0; j < per; ++j) mine += sm.hist[top - j];
    uint32_t total;
    const uint32_t above = block_exclusive_sum<kThreads>(mine, sm.warp, total);
    if (pass == 0 && total <= need) {
      all = true;
      break;
    }
    if (above < need && need <= above + mine) {  // exactly one thread
      uint32_t sum = above;
      int j = 0;
      while (sum + sm.hist[top - j] < need) sum += sm.hist[top - j++];
      sm.digit = static_cast<uint32_t>(top - j);
      sm.above = sum;
      sm.in_bin = sm.hist[top - j];
    }
    __syncthreads();
    prefix |= sm.digit << shift;
    known |= static_cast<uint32_t>(bins - 1) << shift;
    need -= sm.above;
    bin_whole = sm.in_bin == need;
    __syncthreads();
    if (bin_whole) break;  // the whole bin is taken: its lowest key is the border
  }
  // taken: key > border, and the first `need` of key == border
  uint32_t border = prefix;
  if (all || bin_whole) {
    border = all || prefix == 0u ? 0u : prefix - 1u;
    need = 0u;
  }
  constexpr int kItems = 4;
  uint32_t taken = 0u, equal = 0u;
  for (int base = 0; base < n; base += kThreads * kItems) {
    const int i0 = base + tid * kItems;
    uint32_t gt = 0u, eq = 0u;  // a bit per item
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const uint32_t u = i0 + j < n ? key(i0 + j) : 0u;
      if (u > border) gt |= 1u << j;
      else if (u == border && u != 0u) eq |= 1u << j;
    }
    uint32_t total;
    const uint32_t before = block_exclusive_sum<kThreads>(
        static_cast<uint32_t>(__popc(gt) | __popc(eq) << 16), sm.warp, total);
    uint32_t g = taken + (before & 0xffffu), e = equal + (before >> 16);
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      if (gt >> j & 1u) {
        emit(static_cast<int>(g + min(e, need)), i0 + j);
        ++g;
      } else if (eq >> j & 1u) {
        if (e < need) emit(static_cast<int>(g + e), i0 + j);
        ++e;
      }
    }
    taken += total & 0xffffu;
    equal += total >> 16;
  }
  return static_cast<int>(taken + min(equal, need));
}

}  // namespace ifa4
