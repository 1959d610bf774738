// The attention weight that keys gather, and the eviction of the keys with the least from a paged
// cache, for sm_100a.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "ifa4_internal.h"
#include "ifa4_paged.cuh"
#include "ifa4_ptx.cuh"

namespace ifa4 {
namespace mass {

// mass[b, g, j] (+)= sum over rows (t, h) of exp(scale q.k + bias - lse).
//
// S^T = K Q^T on tcgen05: a tile has 128 keys in the TMEM lanes and kN rows (query tokens x heads of
// the group) in the columns, so a key's sum over the rows is a sum over one thread's own registers:
// no shuffles, no atomics, a fixed order.  A CTA works on 256 keys at a time, 128 for each of two
// warpgroups, which read the same tile of rows:
//   warp 0      TMA producer: the K tiles of the pair (paged, 128-byte swizzle) and the ring of Q tiles
//   warp 1      issues the products; scores are double-buffered in TMEM for each warpgroup
//   warp 2      -lse, position and place of the bias of every row of a Q tile, beside it in the ring
//   warps 4-..  exponentials and sums; the lane's key stays, the rows stream by (8 warps, 16 where
//               kN is 128, each tile's columns in two halves)
// A sequence whose rows fit one tile keeps it in shared memory while the keys stream by (a few tokens:
// bound by HBM, 256 bytes a key); otherwise the keys stay and the rows stream by (prompts: bound by
// the exponentials and what issues them).  Tiles of rows that all see a key tile, and none of them
// through the bias, take a path without checks; so do chunks of 16 rows that all have a bias.
// 32k tokens causal, 32 heads on 8: 5.0 ms with rel_extent 64 (883 TFLOP/s; the exponentials alone 3.8 to
// 4.1), 6.0 ms with 1024 (5.8 to 6.5 by the power cap).  Counters at 5.2 ms: SFU 68 % busy, tensor
// cores 35 %, issue slots 55 %.
constexpr int kKeys = 128;
constexpr uint32_t kKHalf = kKeys * 128;       // 64 dims of a K tile
constexpr uint32_t kKTile = 2 * kKHalf;        // 128 keys x 256 B
constexpr float kLog2e = 1.4426950408889634f;

constexpr uint32_t kBarBytes = 2560;

// x log2(e) rounded once: the error of a row's lse is one of all its weights, which no sum over the keys
// averages out.
__device__ __forceinline__ float scaled_lse(float x) {
  return static_cast<float>(static_cast<double>(x) * 1.4426950408889634);
}

template <int kN>
struct Layout {
  static constexpr int kKStages = kN >= 128 ? 1 : 2;
  static constexpr int kQStages = kN >= 128 ? 4 : 2;
  static constexpr uint32_t kQHalf = kN * 128;
  static constexpr uint32_t kQTile = 2 * kQHalf;
  static constexpr uint32_t kQ = kKStages * 2 * kKTile;
  static constexpr uint32_t kCols = kQ + kQStages * kQTile;
  static constexpr uint32_t kSums = kCols + kN * 12;
  static constexpr uint32_t kBar = kSums + kQStages * (kN * 8 + 32);
  static constexpr uint32_t kAlloc = kBar + kBarBytes + 1024;
  static constexpr uint32_t kTmemCols = 4 * kN;  // two tiles, two buffers
  // Warpgroups that share a tile's columns: two where the exponentials bound the kernel
  static constexpr int kSplit = kN >= 128 ? 2 : 1;
  static constexpr int kThreads = 128 + kSplit * 256;
  static constexpr int kChunk = kSplit > 1 ? 16 : 32;
};

// Rows of a Q tile: what they all have in common with the rows of every other tile, and their lse.
template <int kN>
struct Columns {
  long long rel[kN];   // element offset of the row's bias at a key from that of the tile's first token
  int token[kN];       // of the tile
};
template <int kN>
struct Sums {
  float nlse[kN];      // -lse * log2(e); -inf: the row adds nothing
  float neg[kN];       // -lse, or -inf too
  uint32_t none[4];    // a bit for every row whose lse is -inf: it adds nothing, whatever its scores are
  uint32_t any_none, unused[3];
};

struct Bars {
  uint64_t k_full[2], k_empty[2], q_full[4], q_empty[4], s_full[2][2], s_empty[2][2], drain;
  uint32_t tmem_base;
  int abort_flag;
  float half[2][2][kKeys];  // sums of the second half of the columns: pair parity, tile, key
};

static_assert(sizeof(Bars) <= kBarBytes, "barrier block");
static_assert(sizeof(Sums<32>) == 32 * 8 + 32 && sizeof(Sums<128>) == 128 * 8 + 32, "room for the sums");

// Tiles of rows that see any of the keys [key0, key0 + 256) of a sequence.
struct Rows {
  int lo, hi;
};
__device__ __forceinline__ Rows rows_of(int key0, int n_q, int n_k, int window, int tokens) {
  const int shift = n_k - n_q;  // position of token 0
  int a = max(0, key0 - shift), z = n_q;
  if (window >= 0) {
    const long long last = static_cast<long long>(key0) + 2 * kKeys - 1 + window - shift;
    if (last + 1 < z) z = static_cast<int>(last + 1 > 0 ? last + 1 : 0);
  }
  if (key0 >= n_k || a >= z) return {0, 0};
  return {a / tokens, (z + tokens - 1) / tokens};
}

__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[16]) { tmem_ld16(addr, r); }
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[32]) { tmem_ld32(addr, r); }

// acc += 2^(scale s + nlse) over a chunk of columns.  All exponentials on the SFU: a share of 1, 2 or 3
// in 8 as polynomials on the FMA pipe (degree 5, 7.5e-8) took 5.18, 5.65 and 5.97 ms where this took 5.19
// (32k prompt, rel_extent 64); a share of 1 or 2 in 16 later 4.83 and 4.92 where this took 4.97, and with
// rel_extent 1024 5.84 and 5.91 where this took 5.88: not worth a second way to the same number.
template <int kC>
__device__ __forceinline__ void add_chunk(const uint32_t (&r)[kC], const float* nlse, uint64_t mul2,
                                          uint64_t (&acc)[2]) {
#pragma unroll
  for (int i = 0; i < kC; i += 4) {
    const float4 nl = *reinterpret_cast<const float4*>(nlse + i);
    float x0, x1, x2, x3;
    f2_unpack(f2_fma(f2_pack(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), mul2,
                     f2_pack(nl.x, nl.y)), x0, x1);
    f2_unpack(f2_fma(f2_pack(__uint_as_float(r[i + 2]), __uint_as_float(r[i + 3])), mul2,
                     f2_pack(nl.z, nl.w)), x2, x3);
    acc[0] = f2_add(acc[0], f2_pack(fast_exp2(x0), fast_exp2(x1)));
    acc[1] = f2_add(acc[1], f2_pack(fast_exp2(x2), fast_exp2(x3)));
  }
}

// A lane's sum over the columns [c0, c_end) of a tile that has rows without an lse among them, which add
// nothing whatever they, the key or the bias hold.  dk and rel_key: distance of the tile's token 0 from
// the key, and its bias there.  Out of line, for tiles that have such rows: a select for every row in the
// loops below cost 3 % of a 32k prompt that has none (6.37 -> 6.59 ms), the test of a tile's flag nothing.
template <int kN>
__device__ __noinline__ float sum_beside_none(const Sums<kN>& m, const Columns<kN>& cols, uint32_t t_s,
                                              int c0, int c_end, int dk, int window, int rel_extent,
                                              const uint16_t* rel_key, float scale_log2) {
  float sum = 0.f;
  for (; c0 < c_end; c0 += 16) {
    uint32_t r[16];
    tmem_load(t_s + c0, r);
    tmem_wait_ld();
    const uint32_t none = m.none[c0 >> 5] >> (c0 & 31);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int d = dk + cols.token[c0 + i];
      const bool seen = c0 + i < c_end && (none >> i & 1u) == 0u &&
                        static_cast<unsigned>(d) <= static_cast<unsigned>(window);
      uint16_t bias = 0;
      load_if(bias, rel_key + cols.rel[c0 + i], seen && d < rel_extent);
      const float y = fast_exp2(__fmaf_rn(__uint_as_float(r[i]), scale_log2,
                                          (bf16_bits_to_float(bias) + m.neg[c0 + i]) * kLog2e));
      sum += seen ? y : 0.f;
    }
  }
  return sum;
}

template <int kN>
__global__ void __launch_bounds__(Layout<kN>::kThreads, 1)
    attention_mass_kernel(const __grid_constant__ AttentionMassKernelArgs a,
                          const __grid_constant__ CUtensorMap tm_q,
                          const __grid_constant__ CUtensorMap tm_k) {
  using L = Layout<kN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + L::kBar);
  Columns<kN>& cols = *reinterpret_cast<Columns<kN>*>(smem + L::kCols);
  Sums<kN>* sums = reinterpret_cast<Sums<kN>*>(smem + L::kSums);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // the pair of key tiles is the slowest index: with a prompt the first keys have the most rows, and
  // the CTAs of all heads with the most rows start first
  const int kvh = blockIdx.x;
  const int b = blockIdx.y;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kKStages; ++i) {
      mbar_init(&bars->k_full[i], 1);
      mbar_init(&bars->k_empty[i], 1);
    }
    for (int i = 0; i < L::kQStages; ++i) {
      mbar_init(&bars->q_full[i], 2);   // TMA and warp 2
      mbar_init(&bars->q_empty[i], 1 + 8 * L::kSplit);  // the products and the summing warps
    }
    for (int w = 0; w < 2; ++w)
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bars->s_full[w][i], 1);
        mbar_init(&bars->s_empty[w][i], 4 * L::kSplit);
      }
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
  }
  if (warp == 3) {
    tmem_alloc(&bars->tmem_base, L::kTmemCols);
    tmem_relinquish();
  }
  const int q0 = __ldg(a.s.cu_q + b);
  int n_q = __ldg(a.s.cu_q + b + 1) - q0;
  if (!IFA4_DBG_CHECK(a.status, n_q <= 0 || (q0 >= 0 && n_q <= a.total_q - q0))) n_q = 0;
  const int n_k = __ldg(a.s.cu_k + b + 1) - __ldg(a.s.cu_k + b);
  const int n_out = min(n_k, a.mass_width);  // keys with a place
  const int n_pairs = ((a.accumulate ? n_out : a.mass_width) + 2 * kKeys - 1) / (2 * kKeys);
  const int tokens = a.tokens_per_tile;
  const bool resident = n_q <= tokens;  // one tile of rows: loaded once
  const int shift = n_k - n_q;
  for (int r = threadIdx.x; r < kN; r += L::kThreads) {
    const int tok = r / a.group;
    cols.token[r] = tok;
    cols.rel[r] = static_cast<long long>(tok) * (a.rel_st + 1) +
                  static_cast<long long>(kvh * a.group + r - tok * a.group) * a.rel_sh;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = bars->tmem_base;
  const AbortCtx ab{&bars->abort_flag, a.status, kStatusDecodeTimeout};

  // of the 96 registers that each of 640 threads starts with, the summing warps take 104 and the
  // others keep 64: together the 61440 of the launch (fewer spills: 7.08 -> 6.82 ms;
  // 112 and 32 the same)
  if (L::kSplit > 1 && warp < 4) setmaxnreg_dec<64>();
  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    const uint64_t pol_k = resident ? l2_policy_evict_first() : l2_policy_evict_last();
    const uint64_t pol_q = l2_policy_evict_last();
    const int box = 1 << a.box_shift;
    const int units = 2 * kKeys >> a.box_shift;  // of the pair, at most 16
    const int page_mask = (1 << a.s.page_shift) - 1;
    const int32_t* table = table_row(a.s, b);
    const uint32_t q_bytes = 2u * static_cast<uint32_t>(tokens * a.group) * 128u;
    uint32_t nk = 0, nq = 0;
    bool ok = true;
    for (int kp = blockIdx.z; kp < n_pairs && ok; kp += gridDim.z) {
      const Rows rows = rows_of(kp * 2 * kKeys, n_q, n_k, a.window_left, tokens);
      if (rows.lo >= rows.hi) continue;
      const int key = kp * 2 * kKeys + lane * box;
      int page = a.s.num_pages;  // out of range: zeros
      if (lane < units && key < n_k) {
        const int p = page_at(a.s, table, key >> a.s.page_shift);
        if (p >= 0) page = p;
      }
      const uint32_t ks = nk % L::kKStages;
      if (!(ok = mbar_wait_warp(&bars->k_empty[ks], ((nk / L::kKStages) & 1) ^ 1, ab))) break;
      if (lane == 0) mbar_arrive_expect_tx(&bars->k_full[ks], 2 * kKTile);
      __syncwarp();
      if (lane < units && IFA4_DBG_CHECK(a.status, page <= a.s.num_pages && (lane + 1) * box <= 2 * kKeys &&
                                                       (key & page_mask) + box <= page_mask + 1)) {
        const int row = lane * box;  // of the pair
        uint8_t* dst = smem + ks * 2 * kKTile + (row / kKeys) * kKTile + (row % kKeys) * 128;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          tma_load_4d_hint(dst + hf * kKHalf, &tm_k, &bars->k_full[ks], hf * 64, kvh,
                           key & page_mask, page, pol_k);
      }
      ++nk;
      for (int qt = rows.lo; qt < rows.hi && !(resident && nq > 0); ++qt, ++nq) {
        const uint32_t qs = nq % L::kQStages;
        if (!(ok = mbar_wait_warp(&bars->q_empty[qs], ((nq / L::kQStages) & 1) ^ 1, ab))) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars->q_full[qs], q_bytes);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
            tma_load_3d_hint(smem + L::kQ + qs * L::kQTile + hf * L::kQHalf, &tm_q,
                             &bars->q_full[qs], hf * 64, kvh * a.group, q0 + qt * tokens, pol_q);
        }
        __syncwarp();
      }
    }
    if (lane == 0) {  // every issued load has landed before the CTA may exit
      for (uint32_t i = 0; i < L::kKStages && i < nk; ++i) {
        const uint32_t at = nk - 1 - i;
        mbar_wait(&bars->k_full[at % L::kKStages], (at / L::kKStages) & 1, ab);
      }
      for (uint32_t i = 0; i < L::kQStages && i < nq; ++i) {
        const uint32_t at = nq - 1 - i;
        mbar_wait(&bars->q_full[at % L::kQStages], (at / L::kQStages) & 1, ab);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_bf16_f32(kKeys, kN, false);
      uint32_t nk = 0, nq = 0, step = 0;
      bool ok = true;
      for (int kp = blockIdx.z; kp < n_pairs && ok; kp += gridDim.z) {
        const Rows rows = rows_of(kp * 2 * kKeys, n_q, n_k, a.window_left, tokens);
        if (rows.lo >= rows.hi) continue;
        const uint32_t ks = nk % L::kKStages;
        if (!(ok = mbar_wait(&bars->k_full[ks], (nk / L::kKStages) & 1, ab))) break;
        for (int qt = rows.lo; qt < rows.hi; ++qt, ++step) {
          const uint32_t qs = resident ? 0u : nq % L::kQStages;
          if (!(resident && nq > 0)) {
            if (!(ok = mbar_wait(&bars->q_full[qs], (nq / L::kQStages) & 1, ab))) break;
            ++nq;
          }
          const uint32_t buf = step & 1;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            if (!(ok = ok && mbar_wait(&bars->s_empty[w][buf], ((step >> 1) & 1) ^ 1, ab))) break;
            tc_fence_after();
            const uint64_t kd = sdesc_sw128(smem_u32(smem + (ks * 2 + w) * kKTile), 16, 1024);
            const uint64_t qd = sdesc_sw128(smem_u32(smem + L::kQ + qs * L::kQTile), 16, 1024);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              umma_ss(tbase + (w * 2 + buf) * kN,
                      sdesc_advance(kd, (kk >> 2) * kKHalf + (kk & 3) * 32),
                      sdesc_advance(qd, (kk >> 2) * L::kQHalf + (kk & 3) * 32), idesc,
                      kk > 0 ? 1u : 0u);
            umma_commit(&bars->s_full[w][buf]);
          }
          if (!ok) break;
          if (!resident) umma_commit(&bars->q_empty[qs]);
        }
        if (ok) umma_commit(&bars->k_empty[ks]);
        ++nk;
      }
      umma_commit(&bars->drain);  // every issued product completes before TMEM is released
      mbar_wait(&bars->drain, 0, ab);
    }
  } else if (warp == 2) {
    // ---------------------------------------------------------------- the lse of each Q tile's rows
    // fetched a tile ahead: a tile waited for its own loads before (25.5 ms of a 32k
    // prompt, 7.5 with this and with the loads of the biases issued together)
    constexpr int kPer = (kN + 31) / 32;
    float l[kPer];
    const auto fetch = [&](int qt) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int r = lane + 32 * i;
        l[i] = INFINITY;
        if (r < kN) {
          const int tok = cols.token[r];
          if (tok < tokens && qt * tokens + tok < n_q)
            l[i] = __ldg(a.lse + static_cast<long long>(kvh * a.group + r - tok * a.group) * a.lse_sh +
                         static_cast<long long>(q0 + qt * tokens + tok) * a.lse_st);
        }
      }
    };
    uint32_t nq = 0;
    bool ok = true;
    for (int kp = blockIdx.z; kp < n_pairs && ok; kp += gridDim.z) {
      const Rows rows = rows_of(kp * 2 * kKeys, n_q, n_k, a.window_left, tokens);
      if (rows.lo >= rows.hi || (resident && nq > 0)) continue;
      fetch(rows.lo);
      for (int qt = rows.lo; qt < rows.hi; ++qt, ++nq) {
        const uint32_t qs = nq % L::kQStages;
        if (!(ok = mbar_wait_warp(&bars->q_empty[qs], ((nq / L::kQStages) & 1) ^ 1, ab))) break;
        uint32_t any_none = 0u;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int r = lane + 32 * i;
          if (r < kN && IFA4_DBG_CHECK(a.status, qt * tokens < n_q)) {
            const float neg = l[i] == -INFINITY ? -INFINITY : -l[i];  // -inf for +inf, too
            sums[qs].nlse[r] = scaled_lse(neg);
            sums[qs].neg[r] = neg;
          }
          const uint32_t none = __ballot_sync(0xffffffffu, l[i] == -INFINITY);
          any_none |= none;
          if (lane == 0) sums[qs].none[i] = none;
        }
        if (lane == 0) sums[qs].any_none = any_none;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->q_full[qs]);
        if (qt + 1 < rows.hi) fetch(qt + 1);
      }
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- exponentials and sums
    const int w = ((warp - 4) >> 2) & 1;
    const int c_begin = ((warp - 4) >> 3) * (kN / L::kSplit);  // first column of this warpgroup
    const int row = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tbase + (static_cast<uint32_t>((warp & 3) * 32) << 16) + w * 2 * kN;
    const uint64_t mul2 = f2_pack(a.scale_log2, a.scale_log2);
    constexpr int kC = L::kChunk, kW = kN / L::kSplit;
    if (L::kSplit > 1) setmaxnreg_inc<104>();
    const int window = a.window_left < 0 ? 0x7fffffff : a.window_left;
    uint32_t nq = 0, step = 0, pairs = 0;
    bool ok = true;
    for (int kp = blockIdx.z; kp < n_pairs; kp += gridDim.z) {
      const int tile0 = kp * 2 * kKeys + w * kKeys;
      const int key = tile0 + row;
      const Rows rows = rows_of(kp * 2 * kKeys, n_q, n_k, a.window_left, tokens);
      uint64_t acc[2] = {0, 0};
      // Full tiles whose rows all see every key of this tile, and none through the bias: from in_lo on,
      // in_n of them
      int in_lo = 0, in_n = 0;
      if (tokens * a.group == kN) {
        const int past = a.rel_extent + tile0 + kKeys - 1 - shift;  // tokens from here on
        in_lo = past > 0 ? (past + tokens - 1) / tokens : 0;
        int in_end = n_q / tokens;
        if (a.window_left >= 0) {
          const long long last = static_cast<long long>(a.window_left) + tile0 - shift + 1;
          in_end = last < tokens ? 0 : min(in_end, static_cast<int>(min(last / tokens, 1ll << 30)));
        }
        in_n = max(0, in_end - in_lo);
      }
      for (int qt = rows.lo; qt < rows.hi && ok; ++qt, ++step) {
        const uint32_t qs = resident ? 0u : nq % L::kQStages;
        const uint32_t buf = step & 1;
        if (static_cast<unsigned>(qt - in_lo) < static_cast<unsigned>(in_n)) {
          if (!(ok = mbar_wait_warp(&bars->s_full[w][buf], (step >> 1) & 1, ab) &&
                     mbar_wait_warp(&bars->q_full[qs], resident ? 0u : (nq / L::kQStages) & 1, ab)))
            break;
          if (!resident) ++nq;
          tc_fence_after();
          // a sum for each tile, then the sum of those: no long chain of additions to one number
          uint64_t part[2] = {0, 0};
          const float* nlse = &sums[qs].nlse[c_begin];
          const uint32_t t_s = t_lane + buf * kN + c_begin;
          if (sums[qs].any_none != 0u) {
            const int dk = shift + qt * tokens - key;
            part[0] = f2_pack(
                sum_beside_none(sums[qs], cols, t_lane + buf * kN, c_begin, c_begin + kW, dk, window,
                                a.rel_extent,
                                a.rel + static_cast<long long>(q0 + qt * tokens) * a.rel_st + dk,
                                a.scale_log2),
                0.f);
          } else {
            uint32_t r[2][kC];
            tmem_load(t_s, r[0]);
            tmem_wait_ld();
#pragma unroll
            for (int c0 = 0; c0 < kW; c0 += kC) {
              if (c0 + kC < kW) tmem_load(t_s + c0 + kC, r[(c0 / kC + 1) & 1]);
              add_chunk<kC>(r[(c0 / kC) & 1], nlse + c0, mul2, part);
              if (c0 + kC < kW) tmem_wait_ld();
            }
          }
          acc[0] = f2_add(acc[0], part[0]);
          acc[1] = f2_add(acc[1], part[1]);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&bars->s_empty[w][buf]);
            if (!resident) mbar_arrive(&bars->q_empty[qs]);
          }
          continue;
        }
        const int p0 = shift + qt * tokens;  // position of the tile's first token
        const int n_tok = min(tokens, n_q - qt * tokens), n_cols = n_tok * a.group;
        const int c_end = min(n_cols, c_begin + kW);
        // distance of token 0, and its bias at that distance
        const int dk = p0 - key;
        const uint16_t* rel_key = a.rel + static_cast<long long>(q0 + qt * tokens) * a.rel_st + dk;
        // the biases of a chunk, their loads in flight together; 0 where a row has none
        const auto fetch = [&](int c0, uint16_t (&x)[kC]) {
#pragma unroll
          for (int i = 0; i < kC; ++i) x[i] = 0;
          if (c0 >= c_end) return;
          const int p_lo = p0 + cols.token[c0], p_hi = p0 + cols.token[min(c0 + kC, c_end) - 1];
          if (p_lo - (tile0 + kKeys - 1) >= a.rel_extent || p_hi < tile0) return;
          if (c0 + kC <= c_end && p_hi - tile0 < a.rel_extent && p_lo >= tile0 + kKeys - 1) {
#pragma unroll
            for (int i = 0; i < kC; ++i)  // all have one
              if (IFA4_DBG_CHECK(a.status, static_cast<unsigned>(dk + cols.token[c0 + i]) <
                                               static_cast<unsigned>(a.rel_extent)))
                load_now(x[i], rel_key + cols.rel[c0 + i]);
          } else {
#pragma unroll
            for (int i = 0; i < kC; ++i) {
              const int tok = cols.token[c0 + i];
              load_if(x[i], rel_key + cols.rel[c0 + i],
                      tok < n_tok &&
                          static_cast<unsigned>(dk + tok) < static_cast<unsigned>(a.rel_extent));
            }
          }
        };
        // whether every row sees every key of this tile, and none through the bias
        const bool inside = p0 - (tile0 + kKeys - 1) >= a.rel_extent &&
                            (a.window_left < 0 || p0 + n_tok - 1 - tile0 <= a.window_left);
        uint16_t ahead[kC];
        if (!inside) fetch(c_begin, ahead);
        // the wait on the Q tile makes what warp 2 wrote visible
        if (!(ok = mbar_wait_warp(&bars->q_full[qs], resident ? 0u : (nq / L::kQStages) & 1, ab)))
          break;
        if (!resident) ++nq;
        if (!(ok = mbar_wait_warp(&bars->s_full[w][buf], (step >> 1) & 1, ab))) break;
        tc_fence_after();
        const Sums<kN>& m = sums[qs];
        const uint32_t t_s = t_lane + buf * kN;
        uint64_t part[2] = {0, 0};
        float edge = 0.f;
        int c_next = c_begin;
        if (m.any_none != 0u) {
          edge = sum_beside_none(m, cols, t_s, c_begin, c_end, dk, window, a.rel_extent, rel_key,
                                 a.scale_log2);
          c_next = kN;  // nothing is left
        } else if (inside) {  // the chunks that are full
          uint32_t r[2][kC];
          tmem_load(t_s + c_begin, r[0]);
          tmem_wait_ld();
#pragma unroll
          for (int c0 = 0; c0 < kW; c0 += kC) {
            if (c_begin + c0 + kC > c_end) break;
            if (c0 + kC < kW) tmem_load(t_s + c_begin + c0 + kC, r[(c0 / kC + 1) & 1]);
            add_chunk<kC>(r[(c0 / kC) & 1], &m.nlse[c_begin + c0], mul2, part);
            if (c0 + kC < kW) tmem_wait_ld();
            c_next += kC;
          }
          fetch(c_next, ahead);
        }
#pragma unroll 1
        for (int c0 = c_next; c0 < c_end; c0 += kC) {
          uint16_t bias[kC];
#pragma unroll
          for (int i = 0; i < kC; ++i) bias[i] = ahead[i];
          // positions of the chunk's first and last row
          const int p_lo = p0 + cols.token[c0], p_hi = p0 + cols.token[min(c0 + kC, c_end) - 1];
          uint32_t r[kC];
          tmem_load(t_s + c0, r);
          fetch(c0 + kC, ahead);
          tmem_wait_ld();
          if (p_hi < tile0) continue;  // before every key of the tile
          if (a.window_left >= 0 && p_lo - (tile0 + kKeys - 1) > a.window_left) continue;
          // bias - lse first: either may be at the end of the range
          if (c0 + kC <= c_end && p_lo >= tile0 + kKeys - 1 && p_hi - tile0 <= window) {
#pragma unroll
            for (int i = 0; i < kC; i += 4) {  // every row sees every key
              const float4 neg = *reinterpret_cast<const float4*>(&m.neg[c0 + i]);
              const float nl[4] = {neg.x, neg.y, neg.z, neg.w};
              float y[4];
#pragma unroll
              for (int j = 0; j < 4; ++j)
                y[j] = fast_exp2(__fmaf_rn(__uint_as_float(r[i + j]), a.scale_log2,
                                           (bf16_bits_to_float(bias[i + j]) + nl[j]) * kLog2e));
              part[0] = f2_add(part[0], f2_pack(y[0], y[1]));
              part[1] = f2_add(part[1], f2_pack(y[2], y[3]));
            }
          } else {
#pragma unroll
            for (int i = 0; i < kC; ++i) {
              const int tok = cols.token[c0 + i];
              const float y = fast_exp2(__fmaf_rn(__uint_as_float(r[i]), a.scale_log2,
                                                  (bf16_bits_to_float(bias[i]) + m.neg[c0 + i]) *
                                                      kLog2e));
              const bool seen = tok < n_tok && static_cast<unsigned>(dk + tok) <=
                                                   static_cast<unsigned>(window);
              edge += seen ? y : 0.f;
            }
          }
        }
        acc[0] = f2_add(acc[0], f2_add(part[0], f2_pack(edge, 0.f)));
        acc[1] = f2_add(acc[1], part[1]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars->s_empty[w][buf]);
          if (!resident) mbar_arrive(&bars->q_empty[qs]);
        }
      }
      float s0, s1;
      f2_unpack(f2_add(acc[0], acc[1]), s0, s1);
      float sum = s0 + s1;
      if (L::kSplit > 1) {  // the other half of the columns
        float* other = &bars->half[pairs & 1][w][row];
        if (c_begin > 0) *other = sum;
        asm volatile("bar.sync %0, 256;" ::"r"(1 + w) : "memory");
        if (c_begin == 0) sum += *other;
        ++pairs;
      }
      if (ok && c_begin == 0 && key < a.mass_width &&
          IFA4_DBG_CHECK(a.status, key >= 0 && (a.accumulate == 0 || n_pairs * 2 * kKeys > key))) {
        float* dst = a.mass + static_cast<long long>(b) * a.mass_sb +
                     static_cast<long long>(kvh) * a.mass_sh + key;
        if (!a.accumulate) *dst = key < n_out ? sum : 0.f;
        else if (key < n_out && rows.lo < rows.hi) *dst += sum;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 3) tmem_dealloc(tbase, L::kTmemCols);
}

// The same for sequences of up to 16 rows (single tokens): there is nothing to keep, every key is read
// once, and the rows of all of them are one operand of a warp-level MMA.  Every warp has a ring of its
// own, 16 keys a stage, which one of its lanes refills by TMA as soon as the warp has read a stage: no
// barriers between warps, no start to speak of, and 192 KB in flight on an SM.  Bound by HBM, 256 bytes
// a key.  (8 sequences of 4k to 32k keys, one token each: 62 us on the kernel above, whose CTAs start
// slowly and end in a half-empty wave; 50 us with the keys in registers, 64 KB in flight.)  One wave of
// CTAs shares out what all sequences read, in units of 128 keys of one head, so that lengths do not
// matter: 38 us, 40 a call, 5.7 TB/s; 43 with the same number of CTAs for each sequence, four waves of
// them, and 72 with one.  (Two stages and three CTAs an SM: 44; four warps, three stages, four CTAs: 39;
// six stages, two CTAs: 47.)
constexpr int kStreamWarps = 8;
constexpr int kStreamThreads = kStreamWarps * 32;
constexpr int kUnit = kStreamWarps * 16;  // keys that the warps take together
constexpr int kStreamStages = 3;
constexpr uint32_t kStreamHalf = 16 * 128;            // 16 keys, 64 dims
constexpr uint32_t kStreamStage = 2 * kStreamHalf;
constexpr uint32_t kStreamBar = kStreamWarps * kStreamStages * kStreamStage;
constexpr uint32_t kStreamSmem = kStreamBar + 256 + 1024;
static_assert(kStreamWarps * kStreamStages * 8 + 4 <= 256, "barriers and the flag");

__global__ void __launch_bounds__(kStreamThreads, 2)
    attention_mass_stream_kernel(const __grid_constant__ AttentionMassKernelArgs a,
                                 const __grid_constant__ CUtensorMap tm_k) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, qd = lane & 3;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStreamBar) + warp * kStreamStages;
  int* abort_flag = reinterpret_cast<int*>(smem + kStreamBar + 8 * kStreamWarps * kStreamStages);
  uint8_t* ring = smem + warp * kStreamStages * kStreamStage;
  __shared__ uint32_t sums[kStreamWarps], pre[kStreamThreads + 1];
  const int kvh = blockIdx.y;
  if (lane == 0) {
    for (int i = 0; i < kStreamStages; ++i) mbar_init(&full[i], 1);
    if (warp == 0) {
      *abort_flag = 0;
      tma_prefetch_desc(&tm_k);
    }
    fence_mbar_init();
  }
  __syncthreads();
  const AbortCtx ab{abort_flag, a.status, kStatusDecodeTimeout};
  const int mask = (1 << a.s.page_shift) - 1;
  const uint64_t pol = l2_policy_evict_first();
  uint32_t done = 0;  // stages read so far: the ring goes on through all sequences
  bool ok = true;

  // What is read of a sequence: from the first key that any row sees to the last that has a place
  struct Sequence {
    int n_k, q0, n_q, n_out, first;
    __device__ __forceinline__ int units() const {
      return n_q > 0 && first < n_out ? ((n_out + kUnit - 1) / kUnit) - first / kUnit : 0;
    }
  };
  const auto sequence = [&](int b) {
    Sequence x;
    x.n_k = __ldg(a.s.cu_k + b + 1) - __ldg(a.s.cu_k + b);
    x.q0 = __ldg(a.s.cu_q + b);
    x.n_q = __ldg(a.s.cu_q + b + 1) - x.q0;
    if (!IFA4_DBG_CHECK(a.status, x.n_q <= 0 || (x.q0 >= 0 && x.n_q <= a.total_q - x.q0))) x.n_q = 0;
    x.n_out = min(x.n_k, a.mass_width);
    x.first = first_key(x.n_k - x.n_q, a.window_left);
    return x;
  };

  // The keys [key_lo, key_hi) of sequence b, as far as they are read; key_lo a multiple of kUnit.
  const auto stretch = [&](int b, int key_lo, int key_hi) {
    const int32_t* table = table_row(a.s, b);
    const Sequence seq = sequence(b);
    const int q0 = seq.q0, first = seq.first, end = min(key_hi, seq.n_out);
    float* mass = a.mass + static_cast<long long>(b) * a.mass_sb +
                  static_cast<long long>(kvh) * a.mass_sh;
    const int shift = seq.n_k - seq.n_q;
    const int n_rows = seq.n_q * a.group;
    int k_first = key_lo + warp * 16;
    if (k_first + 15 < first) k_first += kUnit * ((first - k_first - 15 + kUnit - 1) / kUnit);
    const auto visible = [&](int k0) { return k0 < end; };
    // page of the 16 keys from k0 on (page_size is a multiple of 16); num_pages reads zeros
    const auto page_of = [&](int k0) {
      int page = a.s.num_pages;
      if (visible(k0)) {
        const int p = page_at(a.s, table, k0 >> a.s.page_shift);
        if (p >= 0) page = p;
      }
      return page;
    };
    const auto load = [&](int k0, int page, uint32_t st) {
      if (lane == 0 && visible(k0) && IFA4_DBG_CHECK(a.status, page <= a.s.num_pages && (k0 & 15) == 0)) {
        mbar_arrive_expect_tx(&full[st], kStreamStage);
  #pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          tma_load_4d_hint(ring + st * kStreamStage + hf * kStreamHalf, &tm_k, &full[st], hf * 64, kvh,
                           k0 & mask, page, pol);
      }
    };
    // more than 16 rows (the caller's hint was too small): the keys once more for the next 16
    for (int r0 = 0; (r0 == 0 || r0 < n_rows) && ok; r0 += 16) {
      // the ring's first stages
      int page_next;
      {
        int pages[kStreamStages];
  #pragma unroll
        for (int i = 0; i < kStreamStages; ++i) pages[i] = page_of(k_first + i * kUnit);
        page_next = page_of(k_first + kStreamStages * kUnit);
  #pragma unroll
        for (int i = 0; i < kStreamStages; ++i)
          load(k_first + i * kUnit, pages[i], (done + i) % kStreamStages);
      }
      // the rows: g and g + 8
      uint32_t qa[8][4];
      float lse[2], nlse[2];
      int pos[2];
      const uint16_t* rel[2];
  #pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = r0 + g + 8 * r, tok = row / a.group;
        const bool on = row < n_rows;
        const long long t = q0 + (on ? tok : 0);
        const int h = kvh * a.group + (on ? row - tok * a.group : 0);
        const uint32_t* src = reinterpret_cast<const uint32_t*>(
            a.q + t * a.q_st + static_cast<long long>(h) * a.q_sh);
  #pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          qa[kk][r] = on ? __ldg(src + kk * 8 + qd) : 0u;
          qa[kk][2 + r] = on ? __ldg(src + kk * 8 + 4 + qd) : 0u;
        }
        lse[r] = on ? __ldg(a.lse + h * a.lse_sh + t * a.lse_st) : -INFINITY;
        nlse[r] = lse[r] == -INFINITY ? -INFINITY : scaled_lse(-lse[r]);
        pos[r] = lse[r] == -INFINITY ? -1 : shift + tok;  // a row that adds nothing sees nothing
        rel[r] = a.rel + t * a.rel_st + static_cast<long long>(h) * a.rel_sh;
      }
      const int window = a.window_left < 0 ? 0x7fffffff : a.window_left;
      const int p_min = __reduce_min_sync(0xffffffffu, min(pos[0] < 0 ? 0x7fffffff : pos[0],
                                                           pos[1] < 0 ? 0x7fffffff : pos[1]));
      const int p_max = __reduce_max_sync(0xffffffffu, max(pos[0], pos[1]));

      for (int k0 = k_first; k0 < end; k0 += kUnit) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};  // keys k0 + 8 t + 2 qd + e
        {
          // what the place holds, on its way while the keys are waited for
          float old[2] = {0.f, 0.f};
          const int place = k0 + 8 * g + 2 * qd;
          if (a.accumulate || r0 > 0) {
  #pragma unroll
            for (int e = 0; e < 2; ++e)
              load_plain_if(old[e], mass + place + e, g < 2 && place + e < end);
          }
          const uint32_t st = done % kStreamStages;
          if (!(ok = mbar_wait_warp(&full[st], (done / kStreamStages) & 1, ab))) break;
          const uint32_t base = smem_u32(ring + st * kStreamStage);
          float acc[2][4], half[2][4];  // two halves of the depth, which do not wait for one another
  #pragma unroll
          for (int t = 0; t < 2; ++t)
  #pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = half[t][i] = 0.f;
          {
            const int mi = lane >> 3;  // which 8x8 matrix this lane addresses
            const int row = (mi >> 1) * 8 + (lane & 7);
  #pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
              const int chunk = 2 * kk + (mi & 1);
              uint32_t b0, b1, b2, b3;
              ldsm_x4(base + (chunk >> 3) * kStreamHalf + row * 128 + (((chunk & 7) ^ (row & 7)) << 4),
                      b0, b1, b2, b3);
              mma_bf16(kk & 1 ? half[0] : acc[0], qa[kk], b0, b1);
              mma_bf16(kk & 1 ? half[1] : acc[1], qa[kk], b2, b3);
            }
          }
  #pragma unroll
          for (int t = 0; t < 2; ++t)
  #pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] += half[t][i];
          // the fragment loads have to be done, not only issued, before TMA refills the stage
          fence_proxy_async_smem();
          __syncwarp();
          ++done;
          load(k0 + kStreamStages * kUnit, page_next, st);
          page_next = page_of(k0 + (kStreamStages + 1) * kUnit);
          const bool near = p_min - (k0 + 15) < a.rel_extent;
          if (!near && k0 + 15 <= p_min && p_max - k0 <= window) {
            // every row sees every key, and none through the bias
  #pragma unroll
            for (int t = 0; t < 2; ++t)
  #pragma unroll
              for (int e = 0; e < 2; ++e)
  #pragma unroll
                for (int r = 0; r < 2; ++r) {
                  const float y = fast_exp2(__fmaf_rn(acc[t][2 * r + e], a.scale_log2, nlse[r]));
                  sum[2 * t + e] += pos[r] >= 0 ? y : 0.f;
                }
          } else {
            uint16_t bias[8];
  #pragma unroll
            for (int i = 0; i < 8; ++i) {  // t, e, r
              const int r = i & 1, d = pos[r] - (k0 + 8 * (i >> 2) + 2 * qd + (i >> 1 & 1));
              bias[i] = 0;
              load_if(bias[i], rel[r] + d, pos[r] >= 0 && d >= 0 && d < a.rel_extent);
            }
  #pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = i & 1, t = i >> 2, e = i >> 1 & 1;
              const int d = pos[r] - (k0 + 8 * t + 2 * qd + e);
              // bias - lse first: either may be at the end of the range
              const float y = fast_exp2(__fmaf_rn(bf16_bits_to_float(bias[i]) - lse[r], kLog2e,
                                                  acc[t][2 * r + e] * a.scale_log2));
              sum[2 * t + e] += pos[r] >= 0 && d >= 0 && d <= window ? y : 0.f;
            }
          }
  #pragma unroll
          for (int i = 0; i < 4; ++i) {
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 4);
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 8);
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 16);
          }
  #pragma unroll
          for (int t = 0; t < 2; ++t)
  #pragma unroll
            for (int e = 0; e < 2; ++e)
              if (g == t) sum[2 * t + e] += old[e];
        }
        // lane qd of the first quad has keys 2 qd, 2 qd + 1 of the first eight; the second of the others
        if (g < 2) {
  #pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = k0 + 8 * g + 2 * qd + e;
            const float y = g == 0 ? sum[e] : sum[2 + e];
            if (key < end && IFA4_DBG_CHECK(a.status, key >= key_lo && key < a.mass_width)) mass[key] = y;
          }
        }
      }
    }
  };

  // The units of all sequences in a row, an equal share of them for every CTA of a head
  const auto units = [&](int b) {
    return b < a.s.batch ? static_cast<uint32_t>(sequence(b).units()) : 0u;
  };
  const int tid = threadIdx.x;
  uint32_t total = 0, sum, before = 0, mine = 0;
  for (int b0 = 0; b0 < a.s.batch; b0 += kStreamThreads) {
    mine = units(b0 + tid);
    before = block_exclusive_sum<kStreamThreads>(mine, sums, sum);
    total += sum;
  }
  const uint32_t lo = static_cast<uint32_t>(static_cast<uint64_t>(total) * blockIdx.x / gridDim.x);
  const uint32_t hi = static_cast<uint32_t>(static_cast<uint64_t>(total) * (blockIdx.x + 1) / gridDim.x);
  uint32_t base = 0;
  for (int b0 = 0; b0 < a.s.batch && base < hi; b0 += kStreamThreads) {
    if (a.s.batch > kStreamThreads) {
      mine = units(b0 + tid);
      before = block_exclusive_sum<kStreamThreads>(mine, sums, sum);
    }
    pre[tid] = base + before;
    if (tid == kStreamThreads - 1) pre[kStreamThreads] = base + sum;
    base += sum;
    // the first sequence that does not end before the share
    const int i0 = __syncthreads_count(pre[tid] + mine <= lo);
    for (int i = i0; i < kStreamThreads && pre[i] < hi && ok; ++i) {
      if (pre[i + 1] == pre[i]) continue;
      const int u0 = sequence(b0 + i).first / kUnit;
      stretch(b0 + i, (static_cast<int>(max(lo, pre[i]) - pre[i]) + u0) * kUnit,
              (static_cast<int>(min(hi, pre[i + 1]) - pre[i]) + u0) * kUnit);
    }
    __syncthreads();
  }
  if (!a.accumulate)  // places that no warp above wrote: of keys that no row sees, and behind the keys
    for (int b = 0; b < a.s.batch; ++b) {
      const Sequence seq = sequence(b);
      float* mass = a.mass + static_cast<long long>(b) * a.mass_sb +
                    static_cast<long long>(kvh) * a.mass_sh;
      const int step = static_cast<int>(gridDim.x) * kStreamThreads;
      for (int key = static_cast<int>(blockIdx.x) * kStreamThreads + tid; key < a.mass_width; key += step)
        if (key >= seq.n_out || seq.units() == 0 || (key | 15) < seq.first) mass[key] = 0.f;
    }
  // after a wait that was given up: what is in flight has landed before the memory goes
  if (!ok && lane == 0)
    for (uint32_t i = 0; i < kStreamStages; ++i)
      mbar_wait(&full[(done + i) % kStreamStages], ((done + i) / kStreamStages) & 1, ab);
}

template <int kN>
cudaError_t launch(const AttentionMassKernelArgs& args, const CUtensorMap& tm_q,
                   const CUtensorMap& tm_k, int key_blocks, cudaStream_t stream) {
  static std::atomic<bool> attr[64];
  cudaError_t e = set_smem_limit_once(attention_mass_kernel<kN>, Layout<kN>::kAlloc, attr);
  if (e != cudaSuccess) return e;
  attention_mass_kernel<kN><<<dim3(args.kv_heads, args.s.batch, key_blocks), Layout<kN>::kThreads,
                              Layout<kN>::kAlloc, stream>>>(args, tm_q, tm_k);
  return cudaGetLastError();
}

}  // namespace mass

namespace evict {

// ---------------------------------------------------------------------------------------
// What stays
// ---------------------------------------------------------------------------------------
// A block per sequence and KV head: the border of the masses (see select_largest), then the places
// that stay, in order, with their masses.  Rows of up to 4, 12 and 32 masses a thread are held in
// registers (16 x 8 heads, 64 stay, with the move: 4096 masses 13.0 us with 4 a thread, 15.6 with 12, 23.7
// with 32; 6000 to 12288 15.9 to 17.0 with 12, 17.3 to 18.1 with 16, 23.8 to 24.4 with 32; 14000 to 16384
// 18.3 to 18.9 with 16, 24.5 to 25.1 with 32, which the rows there take; 32768 27.8).
constexpr int kSelectThreads = 1024;

__global__ void __launch_bounds__(kSelectThreads)
    kv_evict_select_kernel(const __grid_constant__ KvEvictKernelArgs a) {
  __shared__ SelectSmem<kSelectThreads> sm;
  const int g = blockIdx.x, b = blockIdx.y;
  launch_dependents();
  // the counter and the flags of the move
  if (g == 0 && b == 0 && threadIdx.x < 4) a.ws[threadIdx.x] = 0;
  int* flags = a.ws + 4 + (static_cast<long long>(b) * a.kv_heads + g) * a.stretches;
  for (int i = threadIdx.x; i < a.stretches; i += kSelectThreads) flags[i] = 0;
  if (g == 0 && b == 0 && threadIdx.x == 0) {
    int sum = 0, at = __ldg(a.s.cu_k);
    a.cu_out[0] = 0;
    for (int i = 0; i < a.s.batch; ++i) {
      const int end = __ldg(a.s.cu_k + i + 1);
      sum += max(0, min(end - at, a.budget));
      at = end;
      a.cu_out[i + 1] = sum;
    }
  }
  const int n = max(0, __ldg(a.s.cu_k + b + 1) - __ldg(a.s.cu_k + b));
  const float* mass = a.mass + static_cast<long long>(b) * a.mass_sb +
                      static_cast<long long>(g) * a.mass_sh;
  float* mass_out = a.mass_out + static_cast<long long>(b) * a.mo_sb +
                    static_cast<long long>(g) * a.mo_sh;
  int32_t* kept = a.kept + (static_cast<long long>(b) * a.kv_heads + g) * a.budget;
  const auto keep = [&](int place, int i) {
    if (IFA4_DBG_CHECK(a.status, place >= 0 && place <= i && place < a.budget && i < n)) kept[place] = i;
  };
  // a key from mass_width on has the mass 0; -inf ranks below every other mass, but can be kept
  const auto rank = [&](int i, float x) {
    if (i < a.first || i >= n - a.recent) return kAlways;
    return i < a.mass_width ? max(rank_of(x), 1u) : rank_of(0.f);
  };
  int stay = n;
  if (n <= a.budget) {
    for (int i = threadIdx.x; i < n; i += kSelectThreads) kept[i] = i;
  } else if (const int there = min(n, a.mass_width); n <= kSelectThreads * 4) {
    stay = select_largest<kSelectThreads, 4>(sm, a.status, mass, there, n, a.budget, rank, keep);
  } else if (n <= kSelectThreads * 12) {
    stay = select_largest<kSelectThreads, 12>(sm, a.status, mass, there, n, a.budget, rank, keep);
  } else if (n <= kSelectThreads * 32) {
    stay = select_largest<kSelectThreads, 32>(sm, a.status, mass, there, n, a.budget, rank, keep);
  } else {
    stay = select_largest_long<kSelectThreads>(
        sm, a.status, n, a.budget, [&](int i) { return rank(i, i < there ? __ldg(mass + i) : 0.f); }, keep);
  }
  if (!IFA4_DBG_CHECK(a.status, stay >= 0 && stay <= a.budget)) stay = 0;
  for (int i = stay + threadIdx.x; i < a.budget; i += kSelectThreads) kept[i] = -1;
  __syncthreads();
  // their masses: places are read back so that the loads are independent of one another
  for (int i0 = threadIdx.x; i0 < a.mass_width; i0 += kSelectThreads * 8) {
    float x[8];
    int at[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + j * kSelectThreads;
      at[j] = i < stay ? kept[i] : a.mass_width;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = 0.f;
      load_if(x[j], mass + at[j], at[j] < a.mass_width && IFA4_DBG_CHECK(a.status, at[j] >= 0));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + j * kSelectThreads;
      if (i < a.mass_width) mass_out[i] = x[j];
    }
  }
}

// ---------------------------------------------------------------------------------------
// Its move to the front
// ---------------------------------------------------------------------------------------
// A block moves kMoveRows kept keys of one sequence and KV head: it copies them to shared memory, says
// so, waits until every earlier stretch of the same head whose keys lie where it is about to write has
// said so too, and writes.  Key `place` comes from kept[place] >= place, so only earlier stretches read
// there.  Stretches are handed out in order by a counter: a block waits for blocks that are running and
// wait for nothing themselves before they say so.  Bound by HBM: 512 bytes read and written a key.
// (16 sequences of 32k keys to 8192, 8 KV heads: 187 us, 5.5 TB/s, of a call of 220 with the choice's 35;
// a block per head that went through its keys with barriers took the call to 364.)
constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 64;
constexpr uint32_t kMoveSmem = kMoveRows * 512;  // K and V rows

__device__ __forceinline__ int load_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// Waits until *flag is set, up to timeout_ns after t0; then the status bit is set and it returns false.
__device__ __forceinline__ bool wait_flag(const int* flag, int* status, unsigned long long t0,
                                          unsigned long long timeout_ns = kWaitTimeoutNs) {
  for (uint32_t it = 1; load_acquire(flag) == 0; ++it) {
    if ((it & 255u) == 0 && globaltimer_ns() - t0 > timeout_ns) {
      atomicOr(status, kStatusEvictTimeout);
      return false;
    }
  }
  return true;
}

// The wait on a flag that nothing sets.
__device__ int g_never_set = 0;
__global__ void __launch_bounds__(32) wait_selftest_kernel(int* status, unsigned long long timeout_ns) {
  wait_flag(&g_never_set, status, globaltimer_ns(), timeout_ns);
}

__global__ void __launch_bounds__(kMoveThreads)
    kv_evict_move_kernel(const __grid_constant__ KvEvictKernelArgs a) {
  __shared__ __align__(16) uint8_t rows[kMoveSmem];
  __shared__ int ticket[2];
  const int heads = a.s.batch * a.kv_heads, total = heads * a.stretches;
  const int mask = (1 << a.s.page_shift) - 1;
  const int part = threadIdx.x & 15, sub = threadIdx.x >> 4;  // 16 bytes of 16 rows at a time
  constexpr int kStep = kMoveThreads / 16, kTurns = kMoveRows / kStep;
  wait_previous_kernel();
  if (threadIdx.x == 0) ticket[0] = atomicAdd(a.ws, 1);
  __syncthreads();
  // what a stretch moves: the pages and places its rows come from and go to (page -1: none)
  int c, bg, from[kTurns], page_from[kTurns], page_to[kTurns];
  const auto plan = [&](int t) {
    c = t / heads;
    bg = t - c * heads;
    const int b = bg / a.kv_heads;
    const int n = __ldg(a.s.cu_k + b + 1) - __ldg(a.s.cu_k + b);
    const int32_t* kept = a.kept + static_cast<long long>(bg) * a.budget;
    const int32_t* table = table_row(a.s, b);
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int place = c * kMoveRows + sub + i * kStep;
      from[i] = n > a.budget && place < a.budget ? kept[place] : place;
    }
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int place = c * kMoveRows + sub + i * kStep;
      page_to[i] = page_from[i] = -1;
      if (from[i] != place && IFA4_DBG_CHECK(a.status, from[i] > place && from[i] < n && place < a.budget &&
                                                           b < a.s.batch && c < a.stretches)) {
        page_to[i] = page_at(a.s, table, place >> a.s.page_shift);
        page_from[i] = page_at(a.s, table, from[i] >> a.s.page_shift);
      }
    }
  };
  int now = 0;
  int t = ticket[0];
  if (t < total) plan(t);
  while (t < total) {
    // the next stretch is taken now, so that its number and its keys are there when this one is done;
    // whoever waits for it waits for this block, which waits for earlier stretches only
    if (threadIdx.x == 0) ticket[now ^ 1] = atomicAdd(a.ws, 1);
    const int g = bg % a.kv_heads;
    bool any = false;
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      if (page_to[i] < 0) continue;
      if (!IFA4_DBG_CHECK(a.status, page_to[i] < a.s.num_pages && page_from[i] < a.s.num_pages)) {
        page_to[i] = -1;
        continue;
      }
      any = true;
      uint8_t* k = rows + (sub + i * kStep) * 512 + part * 16;
      if (page_from[i] >= 0) {
        const long long slot = from[i] & mask;
        cp_async16(smem_u32(k), a.k_cache + page_from[i] * a.k_sp + slot * a.k_st + g * a.k_sh +
                                    part * 8);
        cp_async16(smem_u32(k + 256), a.v_cache + page_from[i] * a.v_sp + slot * a.v_st +
                                          g * a.v_sh + part * 8);
      } else {  // a key without a page is zeros
        *reinterpret_cast<uint4*>(k) = make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4*>(k + 256) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    const int base = c * kMoveRows, this_c = c, this_bg = bg;
    int to[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) to[i] = page_to[i];
    cp_async_wait_all();
    const bool write = __syncthreads_or(any);
    int* flags = a.ws + 4 + static_cast<long long>(this_bg) * a.stretches;
    if (threadIdx.x == 0) {  // this stretch has been read
      __threadfence();
      atomicExch(flags + this_c, 1);
    }
    now ^= 1;
    t = ticket[now];
    if (t < total) plan(t);
    if (write) {
      const int32_t* kept = a.kept + static_cast<long long>(this_bg) * a.budget;
      bool ok = true;
      const unsigned long long t0 = globaltimer_ns();
      for (int e = this_c - 1 - static_cast<int>(threadIdx.x); e >= 0 && ok; e -= kMoveThreads) {
        if (kept[e * kMoveRows + kMoveRows - 1] < base) break;  // and so are all before
        ok = wait_flag(flags + e, a.status, t0);
      }
      if (__syncthreads_or(!ok)) return;
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        if (to[i] < 0) continue;
        const int r = sub + i * kStep;
        const long long slot = (base + r) & mask;
        const uint4* k = reinterpret_cast<const uint4*>(rows + r * 512 + part * 16);
        *reinterpret_cast<uint4*>(a.k_cache + to[i] * a.k_sp + slot * a.k_st + g * a.k_sh +
                                  part * 8) = k[0];
        *reinterpret_cast<uint4*>(a.v_cache + to[i] * a.v_sp + slot * a.v_st + g * a.v_sh +
                                  part * 8) = k[16];
      }
    }
    __syncthreads();  // the ticket's place may be written again
  }
}

}  // namespace evict

static_assert(evict::kMoveRows == kEvictRows, "stretches");

cudaError_t launch_evict_wait_selftest_sm100(int* status, unsigned long long timeout_ns,
                                             cudaStream_t stream) {
  evict::wait_selftest_kernel<<<1, 32, 0, stream>>>(status, timeout_ns);
  return cudaGetLastError();
}

int attention_mass_tile_rows(long long rows, int group) {
  int n = 32;
  while (n < 128 && (n < rows || n < group)) n *= 2;
  return n;
}

cudaError_t launch_attention_mass_stream_sm100(const AttentionMassKernelArgs& args, int blocks,
                                               const CUtensorMap& tm_k, cudaStream_t stream) {
  static std::atomic<bool> attr[64];
  cudaError_t e = set_smem_limit_once(mass::attention_mass_stream_kernel, mass::kStreamSmem, attr);
  if (e != cudaSuccess) return e;
  mass::attention_mass_stream_kernel<<<dim3(blocks, args.kv_heads), mass::kStreamThreads,
                                       mass::kStreamSmem, stream>>>(args, tm_k);
  return cudaGetLastError();
}

cudaError_t launch_attention_mass_sm100(const AttentionMassKernelArgs& args, int tile_rows,
                                        const CUtensorMap& tm_q, const CUtensorMap& tm_k,
                                        int key_blocks, cudaStream_t stream) {
  switch (tile_rows) {
    case 32: return mass::launch<32>(args, tm_q, tm_k, key_blocks, stream);
    case 64: return mass::launch<64>(args, tm_q, tm_k, key_blocks, stream);
    default: return mass::launch<128>(args, tm_q, tm_k, key_blocks, stream);
  }
}

cudaError_t launch_kv_evict_sm100(const KvEvictKernelArgs& args, int blocks, cudaStream_t stream) {
  evict::kv_evict_select_kernel<<<dim3(args.kv_heads, args.s.batch), evict::kSelectThreads, 0,
                                  stream>>>(args);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int total = args.s.batch * args.kv_heads * args.stretches;
  return launch_early(evict::kv_evict_move_kernel, dim3(total < blocks ? total : blocks),
                      evict::kMoveThreads, 0, stream, args);
}

}  // namespace ifa4
