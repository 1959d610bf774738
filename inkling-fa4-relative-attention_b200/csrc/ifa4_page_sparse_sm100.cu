// Sparse attention over the pages of a paged cache, for sm_100a: bounds of a page's keys, scores of
// pages for a query, the choice of pages, and attention over the chosen ones.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "ifa4_internal.h"
#include "ifa4_paged.cuh"
#include "ifa4_ptx.cuh"

namespace ifa4 {
namespace sparse {

__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t x) {
  return *reinterpret_cast<__nv_bfloat162*>(&x);
}
__device__ __forceinline__ uint32_t min_bf162(uint32_t a, uint32_t b) {
  __nv_bfloat162 r = __hmin2_nan(as_bf162(a), as_bf162(b));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max_bf162(uint32_t a, uint32_t b) {
  __nv_bfloat162 r = __hmax2_nan(as_bf162(a), as_bf162(b));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ uint4 min_v4(uint4 a, uint4 b) {
  return make_uint4(min_bf162(a.x, b.x), min_bf162(a.y, b.y), min_bf162(a.z, b.z),
                    min_bf162(a.w, b.w));
}
__device__ __forceinline__ uint4 max_v4(uint4 a, uint4 b) {
  return make_uint4(max_bf162(a.x, b.x), max_bf162(a.y, b.y), max_bf162(a.z, b.z),
                    max_bf162(a.w, b.w));
}
__device__ __forceinline__ uint4 shfl_xor_v4(uint4 v, int m) {
  return make_uint4(__shfl_xor_sync(0xffffffffu, v.x, m), __shfl_xor_sync(0xffffffffu, v.y, m),
                    __shfl_xor_sync(0xffffffffu, v.z, m), __shfl_xor_sync(0xffffffffu, v.w, m));
}

// ---------------------------------------------------------------------------------------
// Bounds of pages
// ---------------------------------------------------------------------------------------
// A warp per page and KV head: half a warp reads a key (16 bytes a lane), eight keys of each half in
// flight; the halves are joined at the end, one writes the minima, the other the maxima (512
// contiguous bytes).  Bound by HBM: 256 bytes a key and head read, 512 a page and head written (8 x 32k
// keys, 8 KV heads: 86 us, 83.5 at the copy rate).
__global__ void __launch_bounds__(kPageBoundsWarps * 32)
    page_bounds_kernel(const __grid_constant__ PageBoundsKernelArgs a) {
  const int lane = threadIdx.x & 31, half = lane >> 4, part = lane & 15;
  const int b = blockIdx.y;
  const int n_q = __ldg(a.s.cu_q + b + 1) - __ldg(a.s.cu_q + b);
  const int n_k = __ldg(a.s.cu_k + b + 1) - __ldg(a.s.cu_k + b);
  if (n_q <= 0 || n_k <= 0) return;
  const int ps = 1 << a.s.page_shift;
  const int c0 = max(0, n_k - n_q) >> a.s.page_shift;
  const int pages = ((n_k - 1) >> a.s.page_shift) - c0 + 1;
  const int32_t* row = table_row(a.s, b);
  const long long units = static_cast<long long>(pages) * a.kv_heads;
  const long long stride = static_cast<long long>(gridDim.x) * kPageBoundsWarps;
  for (long long u = static_cast<long long>(blockIdx.x) * kPageBoundsWarps + (threadIdx.x >> 5);
       u < units; u += stride) {
    const int c = c0 + static_cast<int>(u / a.kv_heads), h = static_cast<int>(u % a.kv_heads);
    const int page = page_at(a.s, row, c);
    if (page < 0) continue;
    const int keys = min(ps, n_k - (c << a.s.page_shift));
    if (!IFA4_DBG_CHECK(a.status, page < a.s.num_pages && h < a.kv_heads && keys >= 1 && keys <= ps))
      continue;
    const uint16_t* src = a.k_cache + static_cast<long long>(page) * a.k_sp +
                          static_cast<long long>(h) * a.k_sh + part * 8;
    uint4 lo, hi;
    lo = hi = *reinterpret_cast<const uint4*>(src);  // key 0 is always there
    for (int r0 = half; r0 < keys; r0 += 16) {
      uint4 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // past the last key: that key once more
        const int r = min(r0 + 2 * i, keys - 1);
        x[i] = *reinterpret_cast<const uint4*>(src + static_cast<long long>(r) * a.k_st);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo = min_v4(lo, x[i]);
        hi = max_v4(hi, x[i]);
      }
    }
    lo = min_v4(lo, shfl_xor_v4(lo, 16));
    hi = max_v4(hi, shfl_xor_v4(hi, 16));
    uint16_t* dst = a.bounds + static_cast<long long>(page) * a.b_sp +
                    static_cast<long long>(h) * a.b_sh + half * 128 + part * 8;
    *reinterpret_cast<uint4*>(dst) = half ? hi : lo;
  }
}

// ---------------------------------------------------------------------------------------
// Scores of pages
// ---------------------------------------------------------------------------------------
// sum_i (max(q_i, 0) max_i + min(q_i, 0) min_i) is a matrix product of depth 256 with the bounds as
// they lie in memory, and runs on warp-level MMAs (16 rows: the heads of a group, of 16 / group
// tokens; 8 pages a warp).  The order of the 128 dims is free as long as both operands have the same:
// lane qd of a quad takes 16 contiguous bytes of every 64 from the bounds as they were copied.  Every
// warp has a ring of its own, eight pages a stage, refilled by 16-byte asynchronous copies as soon as it
// has read a stage.  The largest bias of a page is found by the whole block, 16 keys a thread at a time,
// for the pages within its reach only.  Bound by HBM: 512 bytes a page and head for 16 rows.
// (64 sequences of up to 32k keys: 72 us, 4.9 TB/s.  111 with the bounds loaded straight to registers,
// 104 with the next eight pages loaded ahead, 99 with bulk copies of 512 bytes, which the copy engine
// takes one by one, 105 with blocks that stay and fetch their next piece of work.)
constexpr int kScoreWarps = 4;
constexpr int kScorePages = 256;  // most pages of a block
constexpr int kScoreStages = 2;
// Pages of a stage lie 576 bytes apart: a lane's 16 bytes and those of the seven it reads with are in
// different banks.
constexpr uint32_t kScorePitch = 576;
constexpr uint32_t kScoreStage = 8 * kScorePitch;
constexpr uint32_t kScoreRing = kScoreWarps * kScoreStages * kScoreStage;
constexpr uint32_t kScoreBias = kScoreRing;
constexpr uint32_t kScoreTile = kScoreBias + 16 * kScorePages * 4;
constexpr uint32_t kScoreSmem = kScoreTile + kScoreWarps * 16 * 9 * 4;

__device__ __forceinline__ float max_nan(float x, float y) {  // NaN if either is
  float z;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}

// kHeads: query heads of a KV head, where they are a power of two up to 16 (their largest score is found
// by shuffles); 0: any number, 16 at a time, through shared memory.
template <int kHeads>
__global__ void __launch_bounds__(kScoreWarps * 32, 4)
    page_scores_kernel(const __grid_constant__ PageScoresKernelArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  uint32_t(&bias_rank)[16][kScorePages] =  // largest bias of a row in a page
      *reinterpret_cast<uint32_t(*)[16][kScorePages]>(smem + kScoreBias);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, qd = lane & 3;
  float(&tile)[16][9] = reinterpret_cast<float(*)[16][9]>(smem + kScoreTile)[warp];
  uint8_t* ring = smem + warp * kScoreStages * kScoreStage;
  const int page0 = blockIdx.x * a.block_pages;
  const int kvh = blockIdx.y % a.kv_heads;
  const int rb0 = blockIdx.y / a.kv_heads;
  const int b = blockIdx.z;
  const int width = a.s.table_width, shift = a.s.page_shift;
  const int page1 = min(width, page0 + a.block_pages);
  if (b == a.s.batch) {  // rows of no sequence: in front of the first and behind the last
    const long long first = max(0, __ldg(a.s.cu_q)), end = max(0, __ldg(a.s.cu_q + a.s.batch));
    for (long long i = rb0;; i += a.row_blocks) {
      const long long t = i < first ? i : end + (i - first);
      if (t >= a.total_q) break;
      for (int c = page0 + threadIdx.x; c < page1; c += kScoreWarps * 32)
        a.scores[t * a.sc_st + kvh * a.sc_sh + c] = -INFINITY;
    }
    return;
  }
  const int32_t* table = table_row(a.s, b);
  const int c_warp = page0 + warp * 8;
  constexpr int kStride = kScoreWarps * 8;
  // what a lane copies: 16 bytes of every page (page strides are below 2^32 bytes)
  const uint8_t* bounds_lane =
      reinterpret_cast<const uint8_t*>(a.bounds + static_cast<long long>(kvh) * a.b_sh) + lane * 16;
  const uint32_t page_bytes = static_cast<uint32_t>(a.b_sp * 2);
  const uint32_t ring_lane = smem_u32(ring) + lane * 16;
  uint32_t done = 0;  // stages read so far: the ring goes on through all rounds
  // the pages of the ring's first stages, whatever the lengths turn out to be
  int first_pages[kScoreStages + 1];
#pragma unroll
  for (int i = 0; i <= kScoreStages; ++i) {
    const int c = c_warp + i * kStride + lane;
    first_pages[i] = lane < 8 && c < page1 ? page_at(a.s, table, c) : -1;
  }
  const int q0 = __ldg(a.s.cu_q + b), n_q = __ldg(a.s.cu_q + b + 1) - q0;
  const int n_k = __ldg(a.s.cu_k + b + 1) - __ldg(a.s.cu_k + b);
  if (!IFA4_DBG_CHECK(a.status, n_q <= 0 || (q0 >= 0 && n_q <= a.total_q - q0))) return;
  const int group = kHeads > 0 ? kHeads : a.group;
  const int hb = min(group, 16);            // heads of a row block
  const int tokens = 16 / hb;               // and tokens
  for (int rb = rb0; rb * tokens < n_q; rb += a.row_blocks) {
    const int tok0 = rb * tokens;
    const int n_tok = min(tokens, n_q - tok0);
    const int p0 = n_k - n_q + tok0;  // position of the block's first token
    const int p1 = p0 + n_tok - 1;    // and of its last
    // pages that any token sees
    const int c_lo = first_key(p0, a.window_left) >> shift;
    const int c_hi = p1 >= 0 ? p1 >> shift : -1;
    // eight pages of a warp's turn are read if any of them is seen
    const int c_last = min(c_hi, page1 - 1);
    const auto seen = [&](int c0) { return c0 <= c_last && c0 + 7 >= c_lo; };
    const int lane_page = lane < 8 ? lane : 1 << 28;
    const auto page_of = [&](int c0) {  // of lane's page, lanes 0 to 7; pages that nobody sees are none
      const int c = c0 + lane_page;
      int p = -1;
      if (c >= c_lo && c <= c_last) p = __ldg(table + c);
      return static_cast<unsigned>(p) < static_cast<unsigned>(a.s.num_pages) ? p : -1;
    };
    // Turns in which every row sees all eight pages, without a bias, and none is taken always: from
    // the last token's first pages on (all but the first first_pages) up to those within the bias's
    // reach of the first token
    const int c_inside =
        (first_key(p1, a.window_left) >> shift) + max(1, a.first_pages);
    const int c_inside_end =
        p0 < a.rel_extent || group > 16
            ? -1
            : min(min((p0 - a.rel_extent + 1) >> shift, page1), (p0 >> shift) - a.last_pages + 1) - 8;
    // one group of copies a turn, empty past the last pages; no page: zeros
    const auto load = [&](int c0, int page, uint32_t st) {
      if (seen(c0)) {
        const uint32_t dst = ring_lane + st * kScoreStage;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          int p = __shfl_sync(0xffffffffu, page, i);
          if (!IFA4_DBG_CHECK(a.status, p < a.s.num_pages)) p = -1;
          cp_async16_or_zeros(dst + i * kScorePitch,
                              bounds_lane + static_cast<uint64_t>(static_cast<uint32_t>(max(p, 0))) *
                                                page_bytes,
                              p >= 0);
        }
      }
      cp_async_commit();
    };
    for (int h0 = 0; h0 < group; h0 += 16) {  // one turn for groups of up to 16
      const int n_rows = group <= 16 ? n_tok * hb : min(16, group - h0);
      // row -> token, head
      const auto token_of = [&](int row) { return group <= 16 ? row / hb : 0; };
      const auto head_of = [&](int row, int tok) {
        return kvh * group + (group <= 16 ? row - tok * hb : h0 + row);
      };
      const bool mine = c_lo < page1 && c_hi >= page0;
      int c_first = c_warp;  // the first pages of this warp that are seen
      if (mine && c_first + 7 < c_lo) c_first += (c_lo - c_first - 7 + kStride - 1) / kStride * kStride;
      int page_next;
      {
        int pages[kScoreStages + 1];
        if (c_first == c_warp) {
#pragma unroll
          for (int i = 0; i <= kScoreStages; ++i) pages[i] = first_pages[i];
        } else {
#pragma unroll
          for (int i = 0; i <= kScoreStages; ++i) pages[i] = page_of(c_first + i * kStride);
        }
        page_next = pages[kScoreStages];
#pragma unroll
        for (int i = 0; i < kScoreStages; ++i)
          load(c_first + i * kStride, pages[i], (done + i) % kScoreStages);
      }
      // max(q, 0) and min(q, 0) of rows g and g + 8
      uint4 qp[4][2], qm[4][2];
      int pos[2];
      bool on[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = g + 8 * r, tok = token_of(row);
        on[r] = row < n_rows;
        pos[r] = p0 + tok;
        const uint16_t* src = a.q + (q0 + tok0 + static_cast<long long>(on[r] ? tok : 0)) * a.q_st +
                              static_cast<long long>(on[r] ? head_of(row, tok) : 0) * a.q_sh + qd * 8;
        const uint4 z = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint4 x = z;
          if (mine && on[r]) x = ldg_nc_v4(src + i * 32);
          qp[i][r] = max_v4(x, z);
          qm[i][r] = min_v4(x, z);
        }
      }
      // ---- largest bias of the pages within its reach: the block's keys from `near` on
      const int near = max(max(0, p0 - a.rel_extent + 1), page0 << shift);
      const int slice0 = near >> 4;
      const int slices =
          mine ? (min(p1, ((page1 - 1) << shift) + ((1 << shift) - 1)) >> 4) - slice0 + 1 : 0;
      if (slices > 0) {
        const int c_near = near >> shift;
        const int c_end = min(page1 - 1, c_hi);
        for (int row = 0; row < n_rows; ++row) {
          const int p = p0 + token_of(row);
          for (int c = c_near + static_cast<int>(threadIdx.x); c <= c_end; c += kScoreWarps * 32) {
            int d1 = p - (c << shift);  // the furthest key of the page
            if (a.window_left >= 0) d1 = min(d1, a.window_left);
            if (IFA4_DBG_CHECK(a.status, c >= page0 && c - page0 < kScorePages && row < 16))
              bias_rank[row][c - page0] = d1 >= a.rel_extent ? kRankZero : 0u;
          }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n_rows * slices; i += kScoreWarps * 32) {
          const int row = i / slices, key0 = (slice0 + i - row * slices) << 4;
          const int tok = token_of(row);
          const uint16_t* rel = a.rel + (q0 + tok0 + static_cast<long long>(tok)) * a.rel_st +
                                static_cast<long long>(head_of(row, tok)) * a.rel_sh;
          uint16_t v[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int d = p0 + tok - (key0 + j);
            v[j] = 0xff80u;  // -inf
            load_if(v[j], rel + d, d >= 0 && d < a.rel_extent &&
                                       (a.window_left < 0 || d <= a.window_left));
          }
          uint32_t most = 0u;
#pragma unroll
          for (int j = 0; j < 16; ++j) most = max(most, rank_of(bf16_bits_to_float(v[j])));
          if (most != 0u && IFA4_DBG_CHECK(a.status, static_cast<unsigned>((key0 >> shift) - page0) <
                                                         static_cast<unsigned>(page1 - page0)))
            atomicMax(&bias_rank[row][(key0 >> shift) - page0], most);
        }
        __syncthreads();
      }
      // ---- scores
      // stores the largest over the heads of a token, of all pages that the block has
      const auto store = [&](int tok, int c, float y) {
        if (!IFA4_DBG_CHECK(a.status, q0 + tok0 + tok < a.total_q && c < width)) return;
        float* dst = a.scores + (q0 + tok0 + tok) * a.sc_st + kvh * a.sc_sh + c;
        if (h0 > 0) y = max_nan(*dst, y);  // of the heads before, by the same thread
        if (h0 + 16 >= group && p0 + tok >= 0) {
          const int p = p0 + tok, hi = p >> shift;
          const int lo = first_key(p, a.window_left) >> shift;
          if (c >= lo && c <= hi && (c - lo < a.first_pages || hi - c < a.last_pages)) y = INFINITY;
        }
        *dst = y;
      };
      // where this lane stores the scores of pages 2 qd, 2 qd + 1: the tokens of rows g and g + 8
      constexpr int lanes = kHeads > 8 ? 8 : kHeads > 0 ? kHeads : 1;  // rows of a token among lanes
      int tok_out[2];
      float* out[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int tok = kHeads == 16 ? r : token_of(g + 8 * r);
        tok_out[r] = (g & (lanes - 1)) == 0 && tok < n_tok ? tok : -1;
        out[r] = a.scores + (q0 + tok0 + max(tok_out[r], 0)) * a.sc_st + kvh * a.sc_sh + 2 * qd;
      }
      for (int c0 = c_warp; c0 < page1; c0 += kStride) {
        if (!seen(c0)) {
          for (int i = lane; i < 8 * n_tok; i += 32)
            if (c0 + (i & 7) < page1) store(i >> 3, c0 + (i & 7), -INFINITY);
          continue;
        }
        const uint32_t st = done % kScoreStages;
        cp_async_wait<kScoreStages - 1>();
        __syncwarp();
        float part[4][4];  // four products of depth 64, which do not wait for one another
        const uint8_t* src = ring + st * kScoreStage + g * kScorePitch + qd * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 lo = *reinterpret_cast<const uint4*>(src + i * 64);
          const uint4 hi = *reinterpret_cast<const uint4*>(src + 256 + i * 64);
          const uint32_t pa[4] = {qp[i][0].x, qp[i][1].x, qp[i][0].y, qp[i][1].y};
          const uint32_t pb[4] = {qp[i][0].z, qp[i][1].z, qp[i][0].w, qp[i][1].w};
          const uint32_t ma[4] = {qm[i][0].x, qm[i][1].x, qm[i][0].y, qm[i][1].y};
          const uint32_t mb[4] = {qm[i][0].z, qm[i][1].z, qm[i][0].w, qm[i][1].w};
          if (i == 0) {
            mma_bf16_first(part[0], pa, hi.x, hi.y);
            mma_bf16_first(part[1], pb, hi.z, hi.w);
            mma_bf16_first(part[2], ma, lo.x, lo.y);
            mma_bf16_first(part[3], mb, lo.z, lo.w);
          } else {
            mma_bf16(part[0], pa, hi.x, hi.y);
            mma_bf16(part[1], pb, hi.z, hi.w);
            mma_bf16(part[2], ma, lo.x, lo.y);
            mma_bf16(part[3], mb, lo.z, lo.w);
          }
        }
        __syncwarp();  // the stage has been read
        ++done;
        load(c0 + kScoreStages * kStride, page_next, st);
        page_next = page_of(c0 + (kScoreStages + 1) * kStride);
        float y[4];  // y[2 r + e] is row g + 8 r, page 2 qd + e
#pragma unroll
        for (int i = 0; i < 4; ++i)
          y[i] = ((part[0][i] + part[1][i]) + (part[2][i] + part[3][i])) * a.scale;
        const bool inside = c0 >= c_inside && c0 <= c_inside_end;
        if (!inside) {
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int c = c0 + 2 * qd + e;
              float x = -INFINITY;
              if (on[r] && pos[r] >= 0 && c < page1 && c <= pos[r] >> shift) {
                // distance of the page's nearest key
                const int d0 = max(0, pos[r] - ((c << shift) + ((1 << shift) - 1)));
                if (a.window_left < 0 || d0 <= a.window_left) {
                  x = y[2 * r + e];
                  if (d0 < a.rel_extent &&
                      IFA4_DBG_CHECK(a.status, (c << shift) + ((1 << shift) - 1) >= near))
                    x += value_of(bias_rank[g + 8 * r][c - page0]);
                }
              }
              y[2 * r + e] = x;
            }
        }
        if constexpr (kHeads > 0) {
#pragma unroll
          for (int m = 4; m < 4 * min(kHeads, 8); m *= 2) {
            y[0] = max_nan(y[0], __shfl_xor_sync(0xffffffffu, y[0], m));
            y[1] = max_nan(y[1], __shfl_xor_sync(0xffffffffu, y[1], m));
            if (n_rows > 8) {  // rows 8 to 15 only where there are some
              y[2] = max_nan(y[2], __shfl_xor_sync(0xffffffffu, y[2], m));
              y[3] = max_nan(y[3], __shfl_xor_sync(0xffffffffu, y[3], m));
            }
          }
          if (kHeads == 16) {
            y[0] = max_nan(y[0], y[2]);
            y[1] = max_nan(y[1], y[3]);
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (tok_out[r] < 0) continue;
            if (inside && IFA4_DBG_CHECK(a.status, q0 + tok0 + tok_out[r] < a.total_q &&
                                                       c0 + 2 * qd + 1 < width)) {
              out[r][c0] = y[2 * r];
              out[r][c0 + 1] = y[2 * r + 1];
            } else {
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (c0 + 2 * qd + e < page1) store(tok_out[r], c0 + 2 * qd + e, y[2 * r + e]);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) tile[g + 8 * (i >> 1)][2 * qd + (i & 1)] = y[i];
          __syncwarp();
          const int heads = group <= 16 ? hb : n_rows;
          for (int i = lane; i < 8 * n_tok; i += 32) {
            const int tok = i >> 3, pg = i & 7;
            float x = -INFINITY;
            for (int r = 0; r < heads; ++r) x = max_nan(x, tile[tok * heads + r][pg]);
            if (c0 + pg < page1) store(tok, c0 + pg, x);
          }
          __syncwarp();
        }
      }
      if (rb + a.row_blocks < (n_q + tokens - 1) / tokens || h0 + 16 < group) __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------------------
// Choice of pages
// ---------------------------------------------------------------------------------------
// A block per row and KV head (see select_largest); kItems 0: rows of any length.  Bound by issue slots
// (65 % busy) and the passes' barriers: every element is read once, and its key ranked, binned, counted
// and emitted from registers.  (128 x 8 rows of 8192 pages: 26.7 us with three blocks an SM, 28.7 with
// two, 30.6 with four, which spill; one row of 2048: 5.5, 5.9 and 5.9 a call.)
template <int kThreads, int kItems>
__global__ void __launch_bounds__(kThreads, kThreads == 512 ? 3 : kThreads == 256 ? 4 : 1)
    select_pages_kernel(const __grid_constant__ SelectPagesKernelArgs a) {
  __shared__ SelectSmem<kThreads> sm;
  const int g = blockIdx.y;
  for (long long t = blockIdx.x; t < a.rows; t += gridDim.x) {
    const float* src = a.scores + t * a.sc_st + g * a.sc_sh;
    int32_t* dst = a.pages + t * a.pg_st + g * a.pg_sh;
    const auto emit = [&](int place, int i) {
      if (IFA4_DBG_CHECK(a.status, place >= 0 && place < a.count && i >= 0 && i < a.width)) dst[place] = i;
    };
    int n;
    if constexpr (kItems > 0)
      n = select_largest<kThreads, kItems>(sm, a.status, src, a.width, a.width, a.count,
                                           [](int, float x) { return rank_of(x); }, emit);
    else
      n = select_largest_long<kThreads>(sm, a.status, a.width, a.count,
                                        [&](int i) { return rank_of(__ldg(src + i)); }, emit);
    for (int i = n + threadIdx.x; i < a.count; i += kThreads) dst[i] = -1;
  }
}

// ---------------------------------------------------------------------------------------
// Attention over chosen pages
// ---------------------------------------------------------------------------------------
// The streaming decode with the keys of a list: a CTA takes tiles of 64 keys of one row's list for up
// to 16 query heads of one KV head.  Warp 4 follows the list and the block table and loads the tiles'
// units (min(page_size, 64) rows) by TMA into a ring; warps 0 to 3 take 16 keys of every tile, which
// always lie in one page (page_size >= 16), so a warp reads one list entry per tile.  Units and slices
// without a visible key are neither loaded nor computed.  Bound by HBM: 512 bytes a key and KV head
// (64 rows of 256 pages of 16 keys, 8 KV heads: 180 to 184 us captured, 188 to 194 a call, 5.7 TB/s of the
// listed keys).
constexpr int kTileKeys = 64;
constexpr int kStages = 3;
constexpr int kConsumerWarps = 4;
constexpr int kThreads = (kConsumerWarps + 1) * 32;
constexpr uint32_t kHalf = kTileKeys * 128;   // 64 rows x 128 B
constexpr uint32_t kKVTile = 2 * kHalf;       // 64 keys x 256 B
constexpr uint32_t kStageBytes = 2 * kKVTile;
constexpr uint32_t kSmemBar = kStages * kStageBytes;
constexpr uint32_t kSmemAlloc = kSmemBar + 128 + 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Bars {
  uint64_t full[kStages];
  uint64_t empty[kStages];
  int abort_flag;
  int last;  // last entry of the list with a visible key
};
static_assert(sizeof(Bars) <= 128, "barrier block");

__device__ __forceinline__ uint32_t sw128_addr(uint32_t base, int row, int chunk) {
  return base + (chunk >> 3) * kHalf + row * 128 + ((((chunk & 7) ^ (row & 7))) << 4);
}

// x + bias in log2 units.  A bias at the end of bf16's range passes fp32's there: the sum stays finite,
// so that a row whose keys all have the lowest one is their mean, as the formula says.
__device__ __forceinline__ float add_bias(float x, float bias) {
  const float y = __fmaf_rn(bias, kLog2e, x);
  return isinf(y) && isfinite(bias) && isfinite(x) ? copysignf(3.402823466e38f, y) : y;
}

// Pairs of bf16 numbers whose sums are x and y (not negative): what is above their 16th bit, and the
// rest to 8 bits.  The rest gets 2^-23 of the number besides, so that it is never 0 nor negative where
// the number is not 0: a value of infinity stays one in the sum of the two products.
__device__ __forceinline__ uint32_t split_bf16x2(float x, float y, uint32_t& rest) {
  const uint32_t bx = __float_as_uint(x), by = __float_as_uint(y);
  const float rx = x - __uint_as_float(bx & 0xffff0000u), ry = y - __uint_as_float(by & 0xffff0000u);
  rest = pack_bf16x2(__fmaf_rn(x, 0x1p-23f, rx), __fmaf_rn(y, 0x1p-23f, ry));
  return __byte_perm(bx, by, 0x7632);
}

// kCluster: the num_splits CTAs of a row are a cluster and merge in each other's shared memory.
template <bool kCluster>
__global__ void __launch_bounds__(kThreads, 2)
    decode_pages_kernel(const __grid_constant__ DecodePagesKernelArgs a,
                        const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + kSmemBar);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const long long t = blockIdx.x / a.num_splits;
  const int split = static_cast<int>(blockIdx.x - t * a.num_splits);
  const int head_blocks = (a.group + a.heads_per_cta - 1) / a.heads_per_cta;
  const int kvh = blockIdx.y / head_blocks;
  const int hblk = blockIdx.y % head_blocks;
  const int h0 = kvh * a.group + hblk * a.heads_per_cta;
  const int nh = min(a.heads_per_cta, a.group - hblk * a.heads_per_cta);
  if (!kCluster && a.num_splits > 1) launch_dependents();
  // the list's first entries, on their way while the sequence is looked up
  const int32_t* list = a.pages + t * a.pg_st + kvh * a.pg_sh;
  const int entry0 = threadIdx.x < a.num_selected ? __ldg(list + threadIdx.x) : -1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], kConsumerWarps);
    }
    bars->abort_flag = 0;
    bars->last = -1;
    fence_mbar_init();
  }
  int n_k, pos;
  const int b = find_sequence(a.s, t, n_k, pos);
  if (b < 0) {
    if (kCluster ? split > 0 : a.num_splits > 1) return;  // the merge kernel writes such rows
    if (!a.zero_padding) return;
    for (int i = threadIdx.x; i < nh * 128; i += kThreads)
      a.out[t * a.out_st + static_cast<long long>(h0 + (i >> 7)) * a.out_sh + (i & 127)] = 0;
    if (a.lse != nullptr && threadIdx.x < nh)
      a.lse[static_cast<long long>(h0 + threadIdx.x) * a.lse_sh + t * a.lse_st] = -INFINITY;
    return;
  }
  const int hi = pos + 1;  // visible keys [lo, hi); none where hi <= 0
  const int lo = first_key(pos, a.window_left);
  const int c_lo = lo >> a.s.page_shift, c_hi = hi > 0 ? pos >> a.s.page_shift : -1;
  __syncthreads();
  {
    int last = entry0 >= c_lo && entry0 <= c_hi ? static_cast<int>(threadIdx.x) : -1;
    for (int e = threadIdx.x + kThreads; e < a.num_selected; e += kThreads) {
      const int c = __ldg(list + e);
      if (c >= c_lo && c <= c_hi) last = e;
    }
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0 && last >= 0) atomicMax(&bars->last, last);
  }
  __syncthreads();
  const int last = bars->last;
  const AbortCtx ab{&bars->abort_flag, a.status, kStatusDecodeTimeout};
  const int ps = 1 << a.s.page_shift, page_mask = ps - 1;
  const long long keys = static_cast<long long>(last + 1) << a.s.page_shift;
  const int tiles = static_cast<int>((keys + kTileKeys - 1) / kTileKeys);
  const int per = (tiles + a.num_splits - 1) / a.num_splits;
  const int t_lo = split * per, t_hi = min(tiles, t_lo + per);

  float m_r[2] = {-INFINITY, -INFINITY};
  float l_r[2] = {0.f, 0.f};
  float o[16][4];
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  if (warp == kConsumerWarps) {
    // ---------------------------------------------------------------- TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    const uint64_t pol = l2_policy_evict_first();
    const int box = 1 << a.box_shift;
    const int units = kTileKeys >> a.box_shift;
    const int32_t* table = table_row(a.s, b);
    // page of unit `lane` of a tile: -2 nothing to load, num_pages reads zeros
    auto unit_page = [&](int tile) {
      const long long vk = static_cast<long long>(tile) * kTileKeys + lane * box;
      const int e = static_cast<int>(vk >> a.s.page_shift);
      int page = -2;
      if (lane < units && e <= last && IFA4_DBG_CHECK(a.status, e >= 0 && e < a.num_selected)) {
        const int c = __ldg(list + e);
        if (c >= c_lo && c <= c_hi) {
          const int key0 = (c << a.s.page_shift) + (static_cast<int>(vk) & page_mask);
          if (key0 < hi && key0 + box > lo) {
            page = page_at(a.s, table, c);
            if (page < 0) page = a.s.num_pages;
          }
        }
      }
      return page;
    };
    uint32_t n = 0;
    int page = t_lo < t_hi ? unit_page(t_lo) : -2;
    for (int tile = t_lo; tile < t_hi; ++tile, ++n) {
      const int next = tile + 1 < t_hi ? unit_page(tile + 1) : -2;  // in flight across the wait
      const uint32_t st = n % kStages;
      if (!mbar_wait_warp(&bars->empty[st], ((n / kStages) & 1) ^ 1, ab)) break;
      const uint32_t loads = __popc(__ballot_sync(0xffffffffu, page >= 0));
      if (lane == 0) mbar_arrive_expect_tx(&bars->full[st], loads * box * 512u);
      __syncwarp();
      if (page >= 0 && IFA4_DBG_CHECK(a.status, page <= a.s.num_pages && (lane + 1) * box <= kTileKeys)) {
        uint8_t* base = smem + st * kStageBytes + lane * box * 128;
        const int in_page = static_cast<int>(static_cast<long long>(tile) * kTileKeys + lane * box) &
                            page_mask;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          tma_load_4d_hint(base + hf * kHalf, &tm_k, &bars->full[st], hf * 64, kvh, in_page, page,
                           pol);
          tma_load_4d_hint(base + kKVTile + hf * kHalf, &tm_v, &bars->full[st], hf * 64, kvh,
                           in_page, page, pol);
        }
      }
      page = next;
    }
    if (lane == 0) {  // every issued load has landed before the CTA may exit
      for (uint32_t i = 0; i < kStages && i < n; ++i) {
        const uint32_t at = n - 1 - i;
        mbar_wait(&bars->full[at % kStages], (at / kStages) & 1, ab);
      }
    }
  } else {
    // ---------------------------------------------------------------- consumers
    const int g = lane >> 2;
    const int qd = lane & 3;
    uint32_t qa[8][4];
    const uint32_t* qrow0 = reinterpret_cast<const uint32_t*>(
        a.q + t * a.q_st + static_cast<long long>(h0 + g) * a.q_sh);
    const uint32_t* qrow1 = reinterpret_cast<const uint32_t*>(
        a.q + t * a.q_st + static_cast<long long>(h0 + g + 8) * a.q_sh);
    const bool r0v = g < nh, r1v = g + 8 < nh;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      qa[kk][0] = r0v ? __ldg(qrow0 + kk * 8 + qd) : 0u;
      qa[kk][1] = r1v ? __ldg(qrow1 + kk * 8 + qd) : 0u;
      qa[kk][2] = r0v ? __ldg(qrow0 + kk * 8 + 4 + qd) : 0u;
      qa[kk][3] = r1v ? __ldg(qrow1 + kk * 8 + 4 + qd) : 0u;
    }
    const uint16_t* relr[2];
    relr[0] = a.rel + t * a.rel_st + static_cast<long long>(h0 + g) * a.rel_sh;
    relr[1] = a.rel + t * a.rel_st + static_cast<long long>(h0 + g + 8) * a.rel_sh;
    const int wrow = warp * 16;  // this warp's 16 keys within the tile
    // list entry of this warp's slice
    auto entry = [&](int tile) {
      const long long vk = static_cast<long long>(tile) * kTileKeys + wrow;
      const int e = static_cast<int>(vk >> a.s.page_shift);
      return e <= last && IFA4_DBG_CHECK(a.status, e >= 0 && e < a.num_selected) ? __ldg(list + e) : -1;
    };
    uint32_t n = 0;
    int c = t_lo < t_hi ? entry(t_lo) : -1;
    for (int tile = t_lo; tile < t_hi; ++tile, ++n) {
      const int next = tile + 1 < t_hi ? entry(tile + 1) : -1;
      const uint32_t st = n % kStages;
      if (!mbar_wait_warp(&bars->full[st], (n / kStages) & 1, ab)) break;
      int kt = hi;  // position of the slice's first key
      if (c >= c_lo && c <= c_hi)
        kt = (c << a.s.page_shift) +
             (static_cast<int>(static_cast<long long>(tile) * kTileKeys + wrow) & page_mask);
      c = next;
      if (kt < hi && kt + 16 > lo) {
        const uint32_t kbase = smem_u32(smem + st * kStageBytes);
        const uint32_t vbase = kbase + kKVTile;
        // ---- S = Q K^T for 16 keys (two n8 tiles)
        float s[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
        {
          const int mi = lane >> 3;
          const int krow = wrow + (mi >> 1) * 8 + (lane & 7);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            uint32_t b0, b1, b2, b3;
            ldsm_x4(sw128_addr(kbase, krow, 2 * kk + (mi & 1)), b0, b1, b2, b3);
            mma_bf16(s[0], qa[kk], b0, b1);
            mma_bf16(s[1], qa[kk], b2, b3);
          }
        }
        // ---- scale, bias, mask
        float x[2][2][2];  // [row r][ntile][e]
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            x[0][nt][e] = s[nt][e] * a.scale_log2;
            x[1][nt][e] = s[nt][2 + e] * a.scale_log2;
          }
        if (pos - (kt + 15) < a.rel_extent) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (!(r == 0 ? r0v : r1v)) continue;
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int d = pos - (kt + nt * 8 + 2 * qd + e);
                if (d >= 0 && d < a.rel_extent)
                  x[r][nt][e] = add_bias(x[r][nt][e], bf16_bits_to_float(__ldg(relr[r] + d)));
              }
          }
        }
        // masked keys may hold anything: their scores are replaced and their values zeroed (0 * NaN
        // would reach the sum); this lane's V fragments hold keys 2 qd (+1) and 8 + 2 qd (+1)
        uint32_t vm0 = 0xffffffffu, vm1 = 0xffffffffu;
        if (kt < lo || kt + 16 > hi) {
          vm0 = vm1 = 0u;
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int key = kt + nt * 8 + 2 * qd + e;
              if (key < lo || key >= hi) x[0][nt][e] = x[1][nt][e] = -INFINITY;
              else (nt == 0 ? vm0 : vm1) |= e == 0 ? 0x0000ffffu : 0xffff0000u;
            }
        }
        // ---- online softmax per row
        uint32_t pa[4], pb[4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float mt = fmaxf(fmaxf(x[r][0][0], x[r][0][1]), fmaxf(x[r][1][0], x[r][1][1]));
          mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
          mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
          const float m_new = fmaxf(m_r[r], mt);
          const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_r[r] - m_new);
          const float m_use = m_new == -INFINITY ? 0.f : m_new;
          m_r[r] = m_new;
          const float p00 = fast_exp2(x[r][0][0] - m_use), p01 = fast_exp2(x[r][0][1] - m_use);
          const float p10 = fast_exp2(x[r][1][0] - m_use), p11 = fast_exp2(x[r][1][1] - m_use);
          l_r[r] = l_r[r] * alpha + (p00 + p01 + p10 + p11);
#pragma unroll
          for (int dt = 0; dt < 16; ++dt) {
            o[dt][2 * r] *= alpha;
            o[dt][2 * r + 1] *= alpha;
          }
          // P is two bf16 numbers for the product with V: 2^-15 of it is lost, where one number loses
          // 2^-8, which was half of the output's error (64 rows of 256 pages: 184 us, 182 with one
          // number; the same with more products between the two to the same sums)
          pa[r] = split_bf16x2(p00, p01, pb[r]);
          pa[2 + r] = split_bf16x2(p10, p11, pb[2 + r]);
        }
        __syncwarp();
        {
          const int mi = lane >> 3;
          const int vrow = wrow + (mi & 1) * 8 + (lane & 7);
#pragma unroll
          for (int dt = 0; dt < 16; dt += 2) {
            uint32_t b0, b1, b2, b3;
            ldsm_x4_t(sw128_addr(vbase, vrow, dt + (mi >> 1)), b0, b1, b2, b3);
            b0 &= vm0;
            b1 &= vm1;
            b2 &= vm0;
            b3 &= vm1;
            mma_bf16(o[dt], pa, b0, b1);
            mma_bf16(o[dt + 1], pa, b2, b3);
            mma_bf16(o[dt], pb, b0, b1);
            mma_bf16(o[dt + 1], pb, b2, b3);
          }
        }
      }
      // the fragment loads have to be done, not only issued, before TMA refills the stage
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->empty[st]);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l_r[r] += __shfl_xor_sync(0xffffffffu, l_r[r], 1);
      l_r[r] += __shfl_xor_sync(0xffffffffu, l_r[r], 2);
    }
  }

  // ------------------------------------------------------------------ merge the 4 warps
  __syncthreads();  // all TMA traffic has landed and all stages are consumed
  float* mo = reinterpret_cast<float*>(smem);      // [4][16][128]
  float* mm = mo + kConsumerWarps * 16 * 128;      // [4][16]
  float* ml = mm + kConsumerWarps * 16;            // [4][16]
  if (warp < kConsumerWarps) {
    const int g = lane >> 2, qd = lane & 3;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = g + 8 * r;
      if (row >= nh) break;
      if (qd == 0) {
        mm[warp * 16 + row] = m_r[r];
        ml[warp * 16 + row] = l_r[r];
      }
#pragma unroll
      for (int dt = 0; dt < 16; ++dt) {
        mo[(warp * 16 + row) * 128 + dt * 8 + 2 * qd] = o[dt][2 * r];
        mo[(warp * 16 + row) * 128 + dt * 8 + 2 * qd + 1] = o[dt][2 * r + 1];
      }
    }
  }
  __syncthreads();
  float* part_o = ml + kConsumerWarps * 16;                                  // [16][128]
  float2* part_ml = reinterpret_cast<float2*>(part_o + 16 * 128);            // [16]
  // one warp per row, lanes own 4 of the 128 dims
  for (int row = warp; row < nh; row += kConsumerWarps + 1) {
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kConsumerWarps; ++w) M = fmaxf(M, mm[w * 16 + row]);
    const float base = M == -INFINITY ? 0.f : M;  // no score above -inf: sums are 0, or NaN
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kConsumerWarps; ++w) {
      const float m = mm[w * 16 + row];
      const float f = m == -INFINITY ? (ml[w * 16 + row] == 0.f ? 0.f : 1.f) : fast_exp2(m - base);
      const float4 o4 = reinterpret_cast<const float4*>(mo + (w * 16 + row) * 128)[lane];
      L += ml[w * 16 + row] * f;
      acc.x += o4.x * f;
      acc.y += o4.y * f;
      acc.z += o4.z * f;
      acc.w += o4.w * f;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;  // NaN stays
    const float lse2 = L == 0.f ? -INFINITY : base + __log2f(L);
    const int h = h0 + row;
    acc.x *= inv;
    acc.y *= inv;
    acc.z *= inv;
    acc.w *= inv;
    if (kCluster) {  // for the merge below
      reinterpret_cast<float4*>(part_o + row * 128)[lane] = acc;
      if (lane == 0) part_ml[row] = make_float2(L == 0.f ? -INFINITY : base, L);
    } else if (!IFA4_DBG_CHECK(a.status, t < a.total_q && h < a.n_heads)) {
      // a bad row or head: nothing is stored
    } else if (a.num_splits == 1) {
      *reinterpret_cast<uint2*>(a.out + t * a.out_st + static_cast<long long>(h) * a.out_sh +
                                lane * 4) =
          make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w));
      if (lane == 0 && a.lse != nullptr)
        a.lse[static_cast<long long>(h) * a.lse_sh + t * a.lse_st] = lse2 * kLn2;
    } else {
      const long long at = (t * a.n_heads + h) * a.num_splits + split;
      reinterpret_cast<float4*>(a.ws_o + at * 128)[lane] = acc;
      if (lane == 0) reinterpret_cast<float2*>(a.ws_ml)[at] = make_float2(L == 0.f ? -INFINITY : base, L);
    }
  }
  if constexpr (kCluster) {
    // The splits of a row are a cluster: each CTA merges some of the rows out of the others' memory
    // (weights L_s 2^(m_s - max m)), with no second kernel and no workspace.
    cluster_sync();
    for (int row = split + warp * a.num_splits; row < nh;
         row += (kConsumerWarps + 1) * a.num_splits) {
      float M = -INFINITY, L = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int s = 0; s < a.num_splits; ++s)
        M = fmaxf(M, load_cluster(&part_ml[row].x, s));
      if (M != -INFINITY) {
        for (int s = 0; s < a.num_splits; ++s) {
          const float m = load_cluster(&part_ml[row].x, s), l = load_cluster(&part_ml[row].y, s);
          const float w = m == -INFINITY ? 0.f : l * fast_exp2(m - M);  // NaN stays
          const float4 o4 = load_cluster_v4(part_o + row * 128 + lane * 4, s);
          L += w;
          acc.x += w * o4.x;
          acc.y += w * o4.y;
          acc.z += w * o4.z;
          acc.w += w * o4.w;
        }
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;
      const int h = h0 + row;
      if (!IFA4_DBG_CHECK(a.status, t < a.total_q && h < a.n_heads)) continue;
      *reinterpret_cast<uint2*>(a.out + t * a.out_st + static_cast<long long>(h) * a.out_sh +
                                lane * 4) =
          make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
      if (lane == 0 && a.lse != nullptr)
        a.lse[static_cast<long long>(h) * a.lse_sh + t * a.lse_st] =
            L == 0.f ? -INFINITY : (M + __log2f(L)) * kLn2;
    }
    cluster_sync();  // nobody reads this CTA's memory any more
  }
}

// Merge of num_splits normalised partials through the workspace, for more splits than a cluster has: a
// warp per row and head, weights L_s 2^(m_s - max m).
constexpr int kMergeWarps = 4;
__global__ void __launch_bounds__(kMergeWarps * 32)
    decode_pages_merge_kernel(const __grid_constant__ DecodePagesKernelArgs a) {
  const int lane = threadIdx.x & 31;
  const long long at = static_cast<long long>(blockIdx.x) * kMergeWarps + (threadIdx.x >> 5);
  const long long t = at / a.n_heads;
  const int h = static_cast<int>(at - t * a.n_heads);
  int n_k, pos;
  const bool none = t >= a.total_q || find_sequence(a.s, t, n_k, pos) < 0;
  // warps with nothing to write wait, too: this grid does not end before the one it was launched beside
  wait_previous_kernel();
  if (t >= a.total_q || (none && !a.zero_padding)) return;
  float M = -INFINITY, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (!none) {
    const float2* ml = reinterpret_cast<const float2*>(a.ws_ml) + at * a.num_splits;
    for (int s = 0; s < a.num_splits; ++s) M = fmaxf(M, ml[s].x);
    if (M != -INFINITY) {
      for (int s = 0; s < a.num_splits; ++s) {
        const float2 p = ml[s];
        const float w = p.x == -INFINITY ? 0.f : p.y * fast_exp2(p.x - M);  // NaN stays
        const float4 o4 = reinterpret_cast<const float4*>(a.ws_o + (at * a.num_splits + s) * 128)[lane];
        L += w;
        acc.x += w * o4.x;
        acc.y += w * o4.y;
        acc.z += w * o4.z;
        acc.w += w * o4.w;
      }
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  *reinterpret_cast<uint2*>(a.out + t * a.out_st + static_cast<long long>(h) * a.out_sh + lane * 4) =
      make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  if (lane == 0 && a.lse != nullptr)
    a.lse[static_cast<long long>(h) * a.lse_sh + t * a.lse_st] =
        L == 0.f ? -INFINITY : (M + __log2f(L)) * kLn2;
}

}  // namespace sparse

cudaError_t launch_page_bounds_sm100(const PageBoundsKernelArgs& args, int blocks_per_seq,
                                     cudaStream_t stream) {
  sparse::page_bounds_kernel<<<dim3(blocks_per_seq, args.s.batch), kPageBoundsWarps * 32, 0,
                               stream>>>(args);
  return cudaGetLastError();
}

cudaError_t launch_page_scores_sm100(const PageScoresKernelArgs& args, cudaStream_t stream) {
  const dim3 grid((args.s.table_width + args.block_pages - 1) / args.block_pages,
                  args.kv_heads * args.row_blocks, args.s.batch + (args.zero_padding ? 1 : 0));
  static std::atomic<bool> attr[6][64];
  static void (*const kernels[6])(PageScoresKernelArgs) = {
      sparse::page_scores_kernel<0>, sparse::page_scores_kernel<1>, sparse::page_scores_kernel<2>,
      sparse::page_scores_kernel<4>, sparse::page_scores_kernel<8>, sparse::page_scores_kernel<16>};
  int i = 0;
  for (int k = 1; k < 6; ++k)
    if (args.group == 1 << (k - 1)) i = k;
  cudaError_t e = set_smem_limit_once(kernels[i], sparse::kScoreSmem, attr[i]);
  if (e != cudaSuccess) return e;
  kernels[i]<<<grid, sparse::kScoreWarps * 32, sparse::kScoreSmem, stream>>>(args);
  return cudaGetLastError();
}

cudaError_t launch_select_pages_sm100(const SelectPagesKernelArgs& args, cudaStream_t stream) {
  const long long most = 1 << 20;
  const dim3 grid(static_cast<unsigned>(args.rows < most ? args.rows : most), args.kv_heads);
  // the smallest block whose registers hold a row (128 rows of 16384: 10.0 us, 15.8 in the block for 32768)
  if (args.width <= 2048)
    sparse::select_pages_kernel<256, 8><<<grid, 256, 0, stream>>>(args);
  else if (args.width <= 8192)
    sparse::select_pages_kernel<512, 16><<<grid, 512, 0, stream>>>(args);
  else if (args.width <= 16384)
    sparse::select_pages_kernel<1024, 16><<<grid, 1024, 0, stream>>>(args);
  else if (args.width <= 32768)
    sparse::select_pages_kernel<1024, 32><<<grid, 1024, 0, stream>>>(args);
  else
    sparse::select_pages_kernel<1024, 0><<<grid, 1024, 0, stream>>>(args);
  return cudaGetLastError();
}

cudaError_t launch_decode_pages_sm100(const DecodePagesKernelArgs& args, const CUtensorMap& tm_k,
                                      const CUtensorMap& tm_v, cudaStream_t stream) {
  static std::atomic<bool> attr[64], attr_cluster[64];
  const bool cluster = args.num_splits > 1 && args.ws_o == nullptr;
  const auto kernel =
      cluster ? sparse::decode_pages_kernel<true> : sparse::decode_pages_kernel<false>;
  cudaError_t e = set_smem_limit_once(kernel, sparse::kSmemAlloc, cluster ? attr_cluster : attr);
  if (e != cudaSuccess) return e;
  const int head_blocks = (args.group + args.heads_per_cta - 1) / args.heads_per_cta;
  const dim3 grid(static_cast<unsigned>(args.total_q * args.num_splits),
                  args.kv_heads * head_blocks);
  if (cluster) {
    cudaLaunchAttribute dims;
    dims.id = cudaLaunchAttributeClusterDimension;
    dims.val.clusterDim.x = args.num_splits;
    dims.val.clusterDim.y = dims.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(sparse::kThreads);
    cfg.dynamicSmemBytes = sparse::kSmemAlloc;
    cfg.stream = stream;
    cfg.attrs = &dims;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args, tm_k, tm_v);
  }
  kernel<<<grid, sparse::kThreads, sparse::kSmemAlloc, stream>>>(args, tm_k, tm_v);
  e = cudaGetLastError();
  if (e != cudaSuccess || args.num_splits == 1) return e;
  const long long warps = args.total_q * args.n_heads;
  return launch_early(sparse::decode_pages_merge_kernel,
                      dim3(static_cast<unsigned>((warps + sparse::kMergeWarps - 1) /
                                                 sparse::kMergeWarps)),
                      sparse::kMergeWarps * 32, 0, stream, args);
}

}  // namespace ifa4
