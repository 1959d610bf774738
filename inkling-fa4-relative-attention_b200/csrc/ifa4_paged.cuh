// Shared pieces of the long-context kernels: sequences over a paged cache, and the choice of the
// largest values of a row.
#pragma once

#include <stdint.h>

#include "ifa4_internal.h"
#include "ifa4_ptx.cuh"

namespace ifa4 {

// The first key that position p sees (p may be negative, the window as long as it likes).
__device__ __forceinline__ int first_key(int p, int window_left) {
  return window_left >= 0 && p > window_left ? p - window_left : 0;
}

// Sequence b of row t (cu_q[b] <= t < cu_q[b + 1]), its key count and the row's position; -1 for a row
// of none.  Whole warp; one load for a decode batch (one row a sequence), otherwise 32 places are looked
// at a time (one step for up to 32 sequences, two for 1024) and a load for the lengths follows.
__device__ __forceinline__ int find_sequence(const PagedSeqs& s, long long t, int& n_k, int& pos) {
  const int lane = threadIdx.x & 31;
  const int guess = t < s.batch ? static_cast<int>(t) : s.batch - 1;
  const int32_t ends = lane < 4 ? __ldg(s.cu_q + (lane == 0 ? 0 : lane == 1 ? s.batch : guess + lane - 2))
                                : __ldg(s.cu_k + guess + (lane & 1));
  if (t < __shfl_sync(0xffffffffu, ends, 0) || t >= __shfl_sync(0xffffffffu, ends, 1)) return -1;
  int lo = guess, q_end = __shfl_sync(0xffffffffu, ends, 3);
  n_k = __shfl_sync(0xffffffffu, ends, 5) - __shfl_sync(0xffffffffu, ends, 4);
  if (t < __shfl_sync(0xffffffffu, ends, 2) || t >= q_end) {
    lo = 0;
    int hi = s.batch;  // cu_q[lo] <= t < cu_q[hi]
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32;
      const int at = min(lo + (lane + 1) * step, hi);
      const unsigned le = __ballot_sync(0xffffffffu, at < hi && __ldg(s.cu_q + at) <= t);
      const int n = __popc(le);  // offsets ascend: the first n places
      hi = min(lo + (n + 1) * step, hi);
      lo += n * step;
    }
    q_end = __ldg(s.cu_q + lo + 1);
    n_k = __ldg(s.cu_k + lo + 1) - __ldg(s.cu_k + lo);
  }
  pos = n_k - q_end + static_cast<int>(t);
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
// Order-preserving image of a float: -inf is 0 (never chosen), the zeros are equal, and so are all
// NaN, above +inf; kAlways is above all of them.  (x + 0 is +0 for -0 and the canonical NaN for NaN.)
constexpr uint32_t kAlways = 0xffffffffu;
constexpr uint32_t kLowest = 0x007fffffu;           // bits of -inf with their order
constexpr uint32_t kTop = 0xff800000u - kLowest;    // rank of +inf
constexpr uint32_t kRankNan = 0xffffffffu - kLowest;
constexpr uint32_t kRankZero = 0x80000000u - kLowest;
__device__ __forceinline__ uint32_t rank_of(float x) {
  const uint32_t b = __float_as_uint(__fadd_rn(x, 0.f));
  return (b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u)) - kLowest;
}
__device__ __forceinline__ float value_of(uint32_t rank) {
  const uint32_t u = rank + kLowest;
  return __uint_as_float(u ^ (static_cast<uint32_t>(static_cast<int32_t>(~u) >> 31) | 0x80000000u));
}

constexpr int kSelectBins = 2048;
constexpr int kCandidates = 256;

template <int kThreads>
struct SelectSmem {
  uint32_t hist[kSelectBins];
  uint32_t warp[kThreads / 32], warp_equal[kThreads / 32];
  uint32_t candidate[kCandidates];
  uint32_t digit, above, in_bin, low, high, found, border, need;
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
// Returns how many there are.
// For rows of any length: three passes over digits of 11, 11 and 10 bits find the key of the border, one
// more writes what is above it; each reads the row again, which the caches hold.
template <int kThreads, class Key, class Emit>
__device__ __forceinline__ int select_largest_long(SelectSmem<kThreads>& sm, int* status, int n, int count,
                                                   Key key, Emit emit) {
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
      while (IFA4_DBG_CHECK(status, j < per) && sum + sm.hist[top - j] < need) sum += sm.hist[top - j++];
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

// For rows of up to kThreads * kItems elements, which stay in registers (item j of a lane is element
// 32 (kItems warp + j) + lane).  The bins of the first pass divide the range between the smallest and
// the largest finite element, so that they are about equally full: of the keys, which is logarithmic,
// where all have one sign, and of the values where they have both (the keys of small values of either
// sign would take up most of the bins).  With fixed digits of the exponent a few bins held everything,
// and the counts waited for one another (128 x 8 rows of 8192: 56 us).  A bin of up to kCandidates
// elements is ranked directly; a larger one is divided again.
// The element i is values[i], or -inf from `there` on; key(i, value) ranks it.
template <int kThreads, int kItems, class Key, class Emit>
__device__ __forceinline__ int select_largest(SelectSmem<kThreads>& sm, int* status, const float* values,
                                              int there, int n, int count, Key key, Emit emit) {
  static_assert(kThreads >= kCandidates, "one thread a candidate");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int base = warp * 32 * kItems + lane;
  if (tid == 0) {
    sm.high = sm.found = 0u;
    sm.low = 0xffffffffu;
  }
  uint32_t u[kItems];
  {
    float v[kItems];
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      v[j] = -INFINITY;
      load_if(v[j], values + base + 32 * j, base + 32 * j < there);
    }
    for (int i = tid; i < kSelectBins; i += kThreads) sm.hist[i] = 0u;
#pragma unroll
    for (int j = 0; j < kItems; ++j) u[j] = base + 32 * j < n ? key(base + 32 * j, v[j]) : 0u;
  }
  // smallest (less one, which leaves out the keys 0) and largest of the finite ones (less kTop, which
  // puts those from kTop on below them)
  uint32_t low = 0xffffffffu, high = 0u;
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    low = min(low, u[j] - 1u);
    high = max(high, u[j] - kTop);
  }
  low = __reduce_min_sync(0xffffffffu, low);
  high = __reduce_max_sync(0xffffffffu, high);
  __syncthreads();
  if (lane == 0) {
    atomicMin(&sm.low, low);
    atomicMax(&sm.high, high);
  }
  __syncthreads();
  // where the border lies; keys from kTop on are in the last bin of the first pass
  uint32_t lo = sm.low + 1u, hi = sm.high + kTop, need = static_cast<uint32_t>(count), border = 0u;
  float start = 0.f, scale = 0.f;  // the bins of values, where scale > 0
  if (lo < kRankZero && hi > kRankZero && hi < kTop) {
    start = value_of(lo);
    scale = (kSelectBins - 2) / (value_of(hi) - start);  // 0 where the range is not finite
    if (!(scale < 1e30f)) scale = 0.f;                    // nor where it is next to nothing
  }
  const float offset = -start * scale;
  // Bins ascend with the keys (a product with a positive number and a sum do, rounded too).  Keys from
  // kTop on, NaN among them, are in the last bin, and no finite one is.
  const auto value_bin = [&](uint32_t key) {
    const float x = __fmaf_rn(value_of(key), scale, offset);
    return static_cast<uint32_t>(fminf(x, key < kTop ? kSelectBins - 2.f : kSelectBins - 1.f));
  };
  for (bool first = true;; first = false) {
    const int bits = hi > lo ? 32 - __clz(hi - lo) : 0;
    const int shift = bits > 10 ? bits - 10 : 0;  // at most 1024 bins
    if (!first) {
      for (int i = tid; i < kSelectBins; i += kThreads) sm.hist[i] = 0u;
      __syncthreads();
    }
    const bool values_binned = first && scale > 0.f;
    const auto add = [&](uint32_t bin) {
      if (IFA4_DBG_CHECK(status, bin < kSelectBins)) atomicAdd(&sm.hist[bin], 1u);
    };
    const auto candidate = [&](uint32_t key) {
      const uint32_t at = atomicAdd(&sm.found, 1u);
      if (IFA4_DBG_CHECK(status, at < kCandidates)) sm.candidate[at] = key;
    };
    if (values_binned) {
#pragma unroll
      for (int j = 0; j < kItems; ++j)
        if (u[j] != 0u) add(value_bin(u[j]));
    } else if (first) {
#pragma unroll
      for (int j = 0; j < kItems; ++j)
        if (u[j] != 0u) add(u[j] >= kTop ? kSelectBins - 1 : (u[j] - lo) >> shift);
    } else {
#pragma unroll
      for (int j = 0; j < kItems; ++j)
        if (u[j] >= lo && u[j] <= hi) add((u[j] - lo) >> shift);
    }
    __syncthreads();
    // thread 0 has the highest bins
    constexpr int kPer = kSelectBins / kThreads;
    const int high_bin = kSelectBins - 1 - tid * kPer;
    uint32_t mine = 0u;
#pragma unroll
    for (int j = 0; j < kPer; ++j) mine += sm.hist[high_bin - j];
    uint32_t total;
    const uint32_t above = block_exclusive_sum<kThreads>(mine, sm.warp, total);
    if (first && total <= need) {  // everything that can be taken: above the border 0
      need = 0u;
      break;
    }
    if (above < need && need <= above + mine) {  // exactly one thread
      uint32_t sum = above;
      int j = 0;
      while (IFA4_DBG_CHECK(status, j < kPer) && sum + sm.hist[high_bin - j] < need)
        sum += sm.hist[high_bin - j++];
      sm.digit = static_cast<uint32_t>(high_bin - j);
      sm.above = sum;
      sm.in_bin = sm.hist[high_bin - j];
      sm.low = 0xffffffffu;
      sm.high = 0u;
    }
    __syncthreads();
    const uint32_t in_bin = sm.in_bin, digit = sm.digit;
    need -= sm.above;
    if (first && digit == kSelectBins - 1) {
      lo = kTop;
      hi = 0xffffffffu;
    } else if (values_binned) {
      // the keys of the bin lie among those of three bins (which is more than the rounding of a bin's
      // number can be off): few need their own bin looked up
      const uint32_t from = rank_of(start + (static_cast<float>(digit) - 1.f) / scale);
      const uint32_t to = rank_of(start + (static_cast<float>(digit) + 2.f) / scale);
      low = 0xffffffffu;
      high = 0u;
#pragma unroll
      for (int j = 0; j < kItems; ++j)
        if (u[j] - from <= to - from && u[j] != 0u && u[j] < kTop && value_bin(u[j]) == digit) {
          low = min(low, u[j]);
          high = max(high, u[j]);
          if (in_bin <= kCandidates) candidate(u[j]);
        }
      low = __reduce_min_sync(0xffffffffu, low);
      high = __reduce_max_sync(0xffffffffu, high);
      if (lane == 0 && low <= high) {
        atomicMin(&sm.low, low);
        atomicMax(&sm.high, high);
      }
      __syncthreads();
      lo = sm.low;
      hi = sm.high;
    } else {
      lo += digit << shift;
      hi = min(hi, lo + ((1u << shift) - 1u));
    }
    if (in_bin == need) {  // the whole bin: everything above the key before its first
      border = lo - 1u;
      need = 0u;
      break;
    }
    if (lo == hi) {  // equal keys: the first `need` of them
      border = lo;
      break;
    }
    if (in_bin <= kCandidates) {
      if (!values_binned || digit == kSelectBins - 1) {
#pragma unroll
        for (int j = 0; j < kItems; ++j)
          if (u[j] >= lo && u[j] <= hi) candidate(u[j]);
        __syncthreads();
      }
      if (tid < static_cast<int>(in_bin)) {
        const uint32_t x = sm.candidate[tid];
        uint32_t larger = 0u, equal = 0u;
        for (uint32_t j = 0; j < in_bin; ++j) {
          larger += sm.candidate[j] > x;
          equal += sm.candidate[j] == x;
        }
        if (larger < need && need <= larger + equal) {  // threads of equal keys write the same
          const bool every = need == larger + equal;    // all equal ones: they are above x - 1
          sm.border = every ? x - 1u : x;
          sm.need = every ? 0u : need - larger;
        }
      }
      __syncthreads();
      border = sm.border;
      need = sm.need;
      break;
    }
    __syncthreads();  // everyone has read what the next round writes
  }
  // taken: key > border, and the first `need` of key == border
  uint32_t gt = 0u, eq = 0u;
  if (need == 0u) {  // the keys are not needed any more: which lanes' are above
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      u[j] = __ballot_sync(0xffffffffu, u[j] > border);
      gt += __popc(u[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      gt += __popc(__ballot_sync(0xffffffffu, u[j] > border));
      eq += __popc(__ballot_sync(0xffffffffu, u[j] == border));
    }
  }
  if (lane == 0) {
    sm.warp[warp] = gt;
    sm.warp_equal[warp] = eq;
  }
  __syncthreads();
  constexpr int kWarps = kThreads / 32;
  const uint32_t wg = lane < kWarps ? sm.warp[lane] : 0u, we = lane < kWarps ? sm.warp_equal[lane] : 0u;
  uint32_t g = __reduce_add_sync(0xffffffffu, lane < warp ? wg : 0u);
  uint32_t e = __reduce_add_sync(0xffffffffu, lane < warp ? we : 0u);
  const uint32_t taken = __reduce_add_sync(0xffffffffu, wg) +
                         min(__reduce_add_sync(0xffffffffu, we), need);
  const uint32_t before = (1u << lane) - 1u;
  if (need == 0u) {
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      if (u[j] >> lane & 1u) emit(static_cast<int>(g + __popc(u[j] & before)), base + 32 * j);
      g += __popc(u[j]);
    }
  } else {
#pragma unroll 1
    for (int j = 0; j < kItems; ++j) {
      uint32_t x = 0u;  // u[j] without indexing registers
#pragma unroll
      for (int i = 0; i < kItems; ++i) x = i == j ? u[i] : x;
      const uint32_t bg = __ballot_sync(0xffffffffu, x > border);
      const uint32_t be = __ballot_sync(0xffffffffu, x == border);
      const uint32_t mg = g + __popc(bg & before), me = e + __popc(be & before);
      if (x > border) emit(static_cast<int>(mg + min(me, need)), base + 32 * j);
      else if (x == border && me < need) emit(static_cast<int>(mg + me), base + 32 * j);
      g += __popc(bg);
      e += __popc(be);
    }
  }
  __syncthreads();  // the memory may be used again
  return static_cast<int>(taken);
}

}  // namespace ifa4
