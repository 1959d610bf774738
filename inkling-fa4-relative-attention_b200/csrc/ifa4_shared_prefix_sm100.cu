// Decode attention over a prefix that a batch of sequences shares, for sm_100a: the prefix part
// of ifa4_decode_shared_prefix_launch, and the merge of its partials with those of the
// sequences' own keys (rel_attn_decode_kernel restricted to keys past the prefix).
//
// With G query heads per KV head and B sequences, B * G query rows read the same prefix keys:
// the prefix is a matrix product of up to 128 rows a tile against 128-key tiles, so its K and V
// are read once per 128 (or 256) rows instead of once per sequence, and S = Q K^T and O += P V
// run on tcgen05.  Row r of a tile is head r mod G of sequence r div G; a tile's rows are one TMA
// box of Q ({64 dims, G heads, 128 / G sequences}).
//
// Per row (one softmax thread each): distance d = (len - 1) - key, bias rel[h, d] where
// 0 <= d < R, window d <= W, online softmax in the exp2 domain with P written back to TMEM as
// bf16, exactly as in the prefill kernel (whose roles and TMEM plan this kernel has).
// Precision: scores, maxima, sums (of the unrounded weights) and O are fp32.  P is rounded to bf16
// (2^-8 of a weight at most, of random sign over the keys) because the product wants both operands in
// one 16-bit type and V is bf16, and 2 of 16 exponentials of an interior tile are a polynomial good
// to 7.5e-5, a fiftieth of that rounding.  The outputs' error against 64 bits is 1.3 to 1.4 times that
// of weights in 32 bits (8 behind 2k, 33 behind 10k, 128 behind 32k; the output's own rounding to bf16
// is the larger part of both), the same as the decode's and the prefill's.
// Sequences with fewer keys than the prefix take no part (their rows have weight 0 here; the
// decode kernel then covers all of their keys).
//
// The kernels are launched to overlap: the own keys' kernel starts as soon as the prefix kernel's
// CTAs have, fills the SMs they leave, and merges the prefix's partials into its rows once that
// kernel has completed.  Only when the own keys themselves are split does a third kernel merge all
// partials (its blocks wait for both).
//
// The grid is (row tiles, KV heads, key splits); every CTA writes its rows' normalised fp32
// partial outputs and log2-sum-exps.  The CTA's two softmax groups (and TMEM halves) work on
//   kKeyPair = false: two row tiles at the same keys (batches of more than one tile per KV head:
//                     K and V are shared by 256 rows);
//   kKeyPair = true:  one row tile at alternating key tiles (small batches: one group's softmax
//                     overlaps the other's products; each group writes its own partial).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ifa4_internal.h"
#include "ifa4_ptx.cuh"

namespace ifa4 {
namespace prefix {

constexpr int kBM = 128;
constexpr int kBN = 128;
constexpr int kThreads = 384;
// as in the prefill kernel: warps 0-3 give registers to the eight softmax warps
constexpr int kRegsControl = 56, kRegsSoftmax = 224;
static_assert(4 * 32 * kRegsControl + 8 * 32 * kRegsSoftmax <= 384 * 168, "register split");
constexpr uint32_t kHalf = 128u * 128u;  // 128 rows x 128 B (64 dims)
constexpr uint32_t kTile = 2u * kHalf;
// Q tiles, then the K and V stages: two row tiles and two stages, or one and three.
template <bool kKeyPair>
struct Layout {
  static constexpr int kTiles = kKeyPair ? 1 : 2;
  static constexpr int kStages = kKeyPair ? 3 : 2;
  static constexpr uint32_t kQ = 0;
  static constexpr uint32_t kK = kTiles * kTile;
  static constexpr uint32_t kV = kK + kStages * kTile;
  static constexpr uint32_t kBar = kV + kStages * kTile;
  static constexpr uint32_t kAlloc = kBar + 256 + 1024;  // + slack for 1024-byte alignment
};
static_assert(Layout<true>::kAlloc <= 227u * 1024u && Layout<false>::kAlloc <= 227u * 1024u,
              "shared memory");
constexpr uint32_t kTmemCols = 512;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleThreshold = 8.0f;

constexpr uint32_t kIdescQK = idesc_bf16_f32(128, 128, /*b_mn_major=*/false);
constexpr uint32_t kIdescPV = idesc_bf16_f32(128, 128, /*b_mn_major=*/true);

struct Bars {
  uint64_t q_full;
  uint64_t k_full[3], k_empty[3];
  uint64_t v_full[3], v_empty[3];
  uint64_t s_full[2], p_full[2];
  uint64_t o_full[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
  // Over the CTA's rows that take part: the first visible key (upper half) and, of the sequences
  // that see it, the first (lower half), whose table row names the prefix pages: with a window no
  // other row needs to name all of them still.  All ones: no row takes part.
  unsigned long long first;
};
constexpr unsigned long long kNoRow = ~0ull;
static_assert(sizeof(Bars) <= 256, "barrier block");

// Position in a ring of kStages stages.
template <int kStages>
struct Ring {
  uint32_t stage = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1u;
    }
  }
};

__device__ __forceinline__ void issue_qk(uint32_t tmem_s, uint32_t q_addr, uint32_t k_addr) {
  const uint64_t qd = sdesc_sw128(q_addr, 16, 1024);
  const uint64_t kd = sdesc_sw128(k_addr, 16, 1024);
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) {
    const uint32_t off = (kk >> 2) * kHalf + (kk & 3) * 32;
    umma_ss(tmem_s, sdesc_advance(qd, off), sdesc_advance(kd, off), kIdescQK, kk > 0 ? 1u : 0u);
  }
}

__device__ __forceinline__ void issue_pv(uint32_t tmem_o, uint32_t tmem_p, uint32_t v_addr,
                                         bool accumulate) {
  const uint64_t vd = sdesc_sw128(v_addr, kHalf, 1024);
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    umma_ts(tmem_o, tmem_p + kk * 8, sdesc_advance(vd, kk * 2048), kIdescPV,
            (kk > 0 || accumulate) ? 1u : 0u);
}

// Eight fp32 values of a row of partials, whose offsets in the workspace are multiples of 32 bytes:
// one 32-byte store where the workspace itself starts on such a boundary (`sectors`), two 16-byte
// ones where it is only 16-byte aligned, as the C ABI allows.
__device__ __forceinline__ void store_sector(float* dst, const float (&f)[8], bool sectors) {
  if (sectors) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "f"(f[0]), "f"(f[1]),
                 "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
                 : "memory");
  } else {
    reinterpret_cast<float4*>(dst)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}

// Row r of row tile `tile`: its sequence and head, and whether it takes part.
struct Row {
  int b, h, len;
  bool on;
};
__device__ __forceinline__ Row row_of(const SharedPrefixKernelArgs& a, int tile, int r, int kvh) {
  Row w;
  const int bl = r / a.group;
  w.b = tile * a.seqs_per_tile + bl;
  w.h = kvh * a.group + (r - bl * a.group);
  w.on = bl < a.seqs_per_tile && w.b < a.batch;
  w.len = w.on ? __ldg(a.cu_k + w.b + 1) - __ldg(a.cu_k + w.b) : 0;
  w.on = w.on && w.len >= a.prefix_len;
  return w;
}

template <bool kKeyPair>
__global__ void __launch_bounds__(kThreads, 1)
    shared_prefix_kernel(const __grid_constant__ SharedPrefixKernelArgs a,
                         const __grid_constant__ CUtensorMap tm_q,
                         const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  using L = Layout<kKeyPair>;
  Bars* bars = reinterpret_cast<Bars*>(smem + L::kBar);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int tile0 = kKeyPair ? blockIdx.x : 2 * blockIdx.x;
  const int kvh = blockIdx.y;
  const int split = blockIdx.z;

  launch_dependents();  // the own keys' kernel needs nothing from this one
  const int box_rows = a.seqs_per_tile * a.group;
  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&bars->k_full[i], 1);
      mbar_init(&bars->k_empty[i], 1);
      mbar_init(&bars->v_full[i], 1);
      mbar_init(&bars->v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_full[i], 4);
      mbar_init(&bars->o_full[i], 1);
    }
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    bars->first = kNoRow;
    fence_mbar_init();
    // Q right away: it depends on nothing
    const uint64_t pol_q = l2_policy_evict_first();
    mbar_arrive_expect_tx(&bars->q_full, L::kTiles * 2 * box_rows * 128);
#pragma unroll
    for (int i = 0; i < L::kTiles; ++i)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
        tma_load_3d_hint(smem + L::kQ + i * kTile + hf * kHalf, &tm_q, &bars->q_full, hf * 64,
                         kvh * a.group, (tile0 + i) * a.seqs_per_tile, pol_q);
  }
  if (warp == 2) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  if (warp == 3 && lane == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // rows of the Q tiles that no TMA box covers (group does not divide 128) are zeros
  for (int i = threadIdx.x; i < L::kTiles * 2 * (kBM - box_rows) * 8; i += kThreads) {
    const int c = i & 7, rest = i >> 3;
    const int hf = rest / (kBM - box_rows);
    const int row = box_rows + rest - hf * (kBM - box_rows);
    *reinterpret_cast<uint4*>(smem + L::kQ + hf * kHalf + row * 128 + c * 16) =
        make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  __syncthreads();
  // this thread's row (softmax warps)
  const int s = warp >= 4 ? (warp - 4) >> 2 : 0;
  const int row = (warp & 3) * 32 + lane;
  Row me{0, 0, 0, false};
  int key_lo = 0;
  if (warp >= 4) {
    me = row_of(a, tile0 + (kKeyPair ? 0 : s), row, kvh);
    if (a.window_left >= 0) key_lo = max(0, me.len - 1 - a.window_left);
    if (key_lo >= a.prefix_len) me.on = false;
    const int lo = __reduce_min_sync(0xffffffffu, me.on ? key_lo : 0x7fffffff);
    const int ref = __reduce_min_sync(0xffffffffu, me.on && key_lo == lo ? me.b : 0x7fffffff);
    if (lane == 0 && lo != 0x7fffffff)
      atomicMin(&bars->first, static_cast<unsigned long long>(lo) << 32 | static_cast<unsigned>(ref));
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = bars->tmem_base;
  // this CTA's share of the key tiles
  int j_lo = 0, n_kv = 0;
  if (bars->first != kNoRow) {
    const int first = static_cast<int>(bars->first >> 32) / kBN;
    const int all = (a.prefix_len + kBN - 1) / kBN - first;
    const int per = (all + a.splits - 1) / a.splits;
    j_lo = first + split * per;
    n_kv = max(0, min(per, all - split * per));
  }
  const AbortCtx ab{&bars->abort_flag, a.status, kStatusDecodeTimeout};
  if (warp < 4) setmaxnreg_dec<kRegsControl>();
  else setmaxnreg_inc<kRegsSoftmax>();
  if (warp < 4) {
    if (warp == 0 && n_kv == 0) {
      if (lane == 0) mbar_wait(&bars->q_full, 0, ab);  // Q has landed before the CTA may exit
    } else if (warp == 0) {
      // ---------------------------------------------------------------- TMA producer (warp)
      const uint64_t pol_kv = l2_policy_evict_last();
      const int box = 1 << a.box_shift;
      const int units = kBN >> a.box_shift;
      const int page_mask = (1 << a.page_shift) - 1;
      const int first_key = static_cast<int>(bars->first >> 32);
      const int32_t* bt =
          a.block_table + static_cast<long long>(bars->first & 0xffffffffu) * a.bt_stride;
      // page of unit `lane` of key tile j; -1 past the prefix, before the first visible key (a page
      // that has left every window may hold anything by now) or for an entry outside [0, num_pages)
      auto unit_block = [&](int j) {
        const int key = (j_lo + j) * kBN + lane * box;
        int blk = -1;
        if (lane < units && key < a.prefix_len && key + box > first_key) {
          blk = __ldg(bt + (key >> a.page_shift));
          if (blk < 0 || blk >= a.num_pages) blk = -1;
        }
        return blk;
      };
      bool ok = true;
      int blk = unit_block(0);
      Ring<L::kStages> ring;
      for (int j = 0; j < n_kv && ok; ++j, ring.next()) {
        const int key0 = (j_lo + j) * kBN;
        const int blk_next = j + 1 < n_kv ? unit_block(j + 1) : -1;
        const int in_page = (key0 + lane * box) & page_mask;
        const int page = blk >= 0 ? blk : a.num_pages;  // out of range: TMA writes zeros
        const uint32_t st = ring.stage, ph = ring.phase ^ 1u;
        if (!(ok = mbar_wait_warp(&bars->k_empty[st], ph, ab))) break;
        if (lane == 0) mbar_arrive_expect_tx(&bars->k_full[st], kTile);
        __syncwarp();
        if (lane < units) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
            tma_load_4d_hint(smem + L::kK + st * kTile + hf * kHalf + lane * box * 128, &tm_k,
                             &bars->k_full[st], hf * 64, kvh, in_page, page, pol_kv);
        }
        if (!(ok = mbar_wait_warp(&bars->v_empty[st], ph, ab))) break;
        // the unit in which the prefix ends: its later slots may hold anything, so its V rows are
        // copied here with zeros behind the prefix (P is 0 there, but 0 * NaN is not)
        const int pu = (a.prefix_len < key0 + kBN && (a.prefix_len & (box - 1)) != 0)
                           ? (a.prefix_len - key0) >> a.box_shift : -1;
        uint32_t v_bytes = kTile;
        if (pu >= 0) {
          const int pblk = __shfl_sync(0xffffffffu, blk, pu);
          const int pkey = key0 + pu * box;
          const int nvalid = a.prefix_len - pkey;
          const uint16_t* src = a.v + static_cast<long long>(pblk < 0 ? 0 : pblk) * a.v_sp +
                                static_cast<long long>(pkey & page_mask) * a.v_st +
                                static_cast<long long>(kvh) * a.v_sh;
          uint8_t* dst = smem + L::kV + st * kTile;
#pragma unroll 4
          for (int i = lane; i < box * 16; i += 32) {
            const int r = i >> 4, ch = i & 15;
            uint4 val = make_uint4(0u, 0u, 0u, 0u);
            if (r < nvalid && pblk >= 0) val = ldg_nc_v4(src + static_cast<long long>(r) * a.v_st + ch * 8);
            const int rw = pu * box + r;
            *reinterpret_cast<uint4*>(dst + (ch >> 3) * kHalf + rw * 128 +
                                      (((ch & 7) ^ (rw & 7)) << 4)) = val;
          }
          fence_proxy_async_smem();
          __syncwarp();
          v_bytes -= static_cast<uint32_t>(box) * 256u;
        }
        if (lane == 0) mbar_arrive_expect_tx(&bars->v_full[st], v_bytes);
        __syncwarp();
        if (lane < units && lane != pu) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
            tma_load_4d_hint(smem + L::kV + st * kTile + hf * kHalf + lane * box * 128, &tm_v,
                             &bars->v_full[st], hf * 64, kvh, in_page, page, pol_kv);
        }
        blk = blk_next;
      }
      if (lane == 0) {  // every issued load has landed before the CTA may exit
        mbar_wait(&bars->q_full, 0, ab);
        for (int i = 0; i < L::kStages && i < n_kv; ++i) {
          const int last = n_kv - 1 - i;
          mbar_wait(&bars->k_full[last % L::kStages], (last / L::kStages) & 1, ab);
          mbar_wait(&bars->v_full[last % L::kStages], (last / L::kStages) & 1, ab);
        }
      }
    } else if (warp == 1 && n_kv > 0) {
      // ---------------------------------------------------------------- UMMA issuer
      if (lane == 0) {
        const uint32_t q_addr = smem_u32(smem + L::kQ);
        const uint32_t k_addr = smem_u32(smem + L::kK);
        const uint32_t v_addr = smem_u32(smem + L::kV);
        bool ok = mbar_wait(&bars->q_full, 0, ab);
        if (kKeyPair) {
          // key tile j on half s = j mod 2: S(j + 1) is issued before P(j) is waited for
          Ring<L::kStages> kr, vr;
          auto qk = [&](int j) {
            if (!(ok = ok && mbar_wait(&bars->k_full[kr.stage], kr.phase, ab))) return;
            tc_fence_after();
            issue_qk(tbase + (j & 1) * 128, q_addr, k_addr + kr.stage * kTile);
            umma_commit(&bars->s_full[j & 1]);
            umma_commit(&bars->k_empty[kr.stage]);
            kr.next();
          };
          if (ok) qk(0);
          if (ok && n_kv > 1) qk(1);
          for (int j = 0; j < n_kv && ok; ++j, vr.next()) {
            const int half = j & 1;
            if (!(ok = mbar_wait(&bars->p_full[half], (j >> 1) & 1, ab))) break;
            if (!(ok = mbar_wait(&bars->v_full[vr.stage], vr.phase, ab))) break;
            tc_fence_after();
            issue_pv(tbase + 256 + half * 128, tbase + half * 128, v_addr + vr.stage * kTile, j > 1);
            umma_commit(&bars->v_empty[vr.stage]);
            if (j + 2 < n_kv) qk(j + 2);  // overwrites P(j) in order after its product
            else umma_commit(&bars->o_full[half]);
          }
        } else {
          for (int j = 0; j <= n_kv && ok; ++j) {
            const int st = j & 1, pst = (j - 1) & 1;
            if (j < n_kv && !(ok = mbar_wait(&bars->k_full[st], (j >> 1) & 1, ab))) break;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (j > 0) {  // O_i += P_i V of tile j - 1
                if (!(ok = mbar_wait(&bars->p_full[i], (j - 1) & 1, ab))) break;
                if (i == 0 && !(ok = mbar_wait(&bars->v_full[pst], ((j - 1) >> 1) & 1, ab))) break;
                tc_fence_after();
                issue_pv(tbase + 256 + i * 128, tbase + i * 128, v_addr + pst * kTile, j > 1);
              } else {
                tc_fence_after();
              }
              if (j < n_kv) {  // S_i = Q_i K^T of tile j
                issue_qk(tbase + i * 128, q_addr + i * kTile, k_addr + st * kTile);
                umma_commit(&bars->s_full[i]);
              } else {
                umma_commit(&bars->o_full[i]);
              }
            }
            if (!ok) break;
            if (j < n_kv) umma_commit(&bars->k_empty[st]);
            if (j > 0) umma_commit(&bars->v_empty[pst]);
          }
        }
        umma_commit(&bars->drain);  // every issued MMA completes before TMEM is released
        mbar_wait(&bars->drain, 0, ab);
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tbase + lane_off + s * 128;
    const uint32_t t_o = tbase + lane_off + 256 + s * 128;
    const int key_hi = a.prefix_len;
    const int dmax = me.len - 1;  // bias distance at key 0
    const uint16_t* rel_row = a.rel + static_cast<long long>(me.b) * a.rel_st +
                              static_cast<long long>(me.h) * a.rel_sh;
    constexpr int kStep = kKeyPair ? 2 : 1;
    const int j0 = kKeyPair ? s : 0;
    const int part = kKeyPair ? 2 * split + s : split;  // partial this half writes
    float m_run = -INFINITY, l_run = 0.f;
    uint32_t pc = 0;
    bool ok = true;
    for (int j = j0; j < n_kv && ok; j += kStep) {
      const int k0 = (j_lo + j) * kBN;
      const int bl = dmax - a.rel_extent + 1 - k0;  // first column with bias
      const int bh = dmax - k0;                     // last column with bias (>= 0)
      const int cl = key_lo - k0, ch = key_hi - k0;  // visible columns [cl, ch)
      const bool has_bias = me.on && bl <= 127;
      // rows that take no part are never read back: they need no mask
      const bool has_mask = me.on && (cl > 0 || ch < kBN);
      if (!(ok = mbar_wait_warp(&bars->s_full[s], pc & 1, ab))) break;
      ++pc;
      tc_fence_after();
      bool done = false;
      // Interior tiles after the first: exponentials against the running max, redone below when
      // a score outgrew it (see the prefill kernel).
      if (j > j0 && !__any_sync(0xffffffffu, has_bias || has_mask)) {
        const uint64_t mul2 = f2_pack(a.scale_log2, a.scale_log2);
        const uint64_t neg2 = f2_pack(-m_run, -m_run);
        uint64_t acc[4] = {0, 0, 0, 0};
        uint32_t pk[2][32];
        uint32_t rq[2][16];
        tmem_ld16(t_s, rq[0]);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (c < 7) tmem_ld16(t_s + (c + 1) * 16, rq[(c + 1) & 1]);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int col = c * 16 + 2 * i;
            float y0, y1;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(rq[c & 1][2 * i]),
                                     __uint_as_float(rq[c & 1][2 * i + 1])),
                             mul2, neg2),
                      y0, y1);
            float p0, p1;
            if ((col & 15) < 2) {  // 2 of 16 on the FMA pipe, as in the prefill
              exp2_poly_pair_capped(y0, y1, p0, p1);
            } else {
              p0 = fast_exp2(y0);
              p1 = fast_exp2(y1);
            }
            acc[i & 3] = f2_add(acc[i & 3], f2_pack(p0, p1));
            pk[c >> 2][(c & 3) * 8 + i] = pack_bf16x2(p0, p1);
          }
          if (c < 7) tmem_wait_ld();
        }
        const uint64_t a01 = f2_add(acc[0], acc[1]), a23 = f2_add(acc[2], acc[3]);
        float u0, u1;
        f2_unpack(f2_add(a01, a23), u0, u1);
        const float l_tile = u0 + u1;
        if (__all_sync(0xffffffffu, l_tile <= 4294967296.0f)) {  // false for inf and NaN
          tmem_st32(t_s, pk[0]);
          tmem_st32(t_s + 32, pk[1]);
          l_run += l_tile;
          done = true;
        }
      }
      if (!done) {
        // Pass 1: the logits (scaled, biased, masked) replace S in TMEM; their row max.  The
        // chunk loops stay rolled: a short launch runs them once or twice per CTA, and fetching
        // unrolled code costs it more than the TMEM round trips.
        float mx = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t r[32];
          tmem_ld32(t_s + c * 32, r);
          tmem_wait_ld();
          float x[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]) * a.scale_log2;
          const bool chunk_bias = has_bias && c * 32 + 31 >= bl && c * 32 <= bh;
          if (a.bias_vec) {
            if (__any_sync(0xffffffffu, chunk_bias)) {
              uint32_t win[20];
              load_bias_window(rel_row, bh, c, a.rel_extent, chunk_bias, win);
              add_bias_window(win, bh, c, x);
            }
          } else if (chunk_bias) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int d = bh - c * 32 - i;
              if (d >= 0 && d < a.rel_extent)
                x[i] += bf16_bits_to_float(__ldg(rel_row + d)) * kLog2e;
            }
          }
          if (has_mask) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int col = c * 32 + i;
              if (col < cl || col >= ch) x[i] = -INFINITY;
            }
          }
          float m0 = x[0], m1 = x[1];
#pragma unroll
          for (int i = 2; i < 30; i += 4) {
            m0 = fmax3(m0, x[i], x[i + 1]);
            m1 = fmax3(m1, x[i + 2], x[i + 3]);
          }
          m0 = fmax3(m0, x[30], x[31]);
          mx = fmax3(mx, m0, m1);
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(x[i]);
          __syncwarp();  // reconverge after the per-row branches: tcgen05.st is .aligned
          tmem_st32(t_s + c * 32, r);
        }
        tmem_wait_st();
        const float m_new = fmaxf(m_run, mx);
        float alpha = 1.f;
        bool need_rescale = false;
        if (j == j0) {
          m_run = m_new;
        } else if (m_new > m_run + kRescaleThreshold) {
          alpha = fast_exp2(m_run - m_new);
          need_rescale = true;
          l_run *= alpha;
          m_run = m_new;
        }
        const float m_use = (m_run == -INFINITY) ? 0.f : m_run;
        __syncwarp();
        // Pass 2: p = 2^(x - m), P (bf16) over the first 64 columns of S.
        uint64_t acc[4] = {0, 0, 0, 0};
        const uint64_t neg2 = f2_pack(-m_use, -m_use);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t r[32];
          tmem_ld32(t_s + c * 32, r);
          tmem_wait_ld();
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float y0, y1;
            f2_unpack(f2_add(f2_pack(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), neg2),
                      y0, y1);
            const float p0 = fast_exp2(y0), p1 = fast_exp2(y1);
            acc[i & 3] = f2_add(acc[i & 3], f2_pack(p0, p1));
            pk[i] = pack_bf16x2(p0, p1);
          }
          tmem_st16(t_s + c * 16, pk);
        }
        const uint64_t a01 = f2_add(acc[0], acc[1]), a23 = f2_add(acc[2], acc[3]);
        float u0, u1;
        f2_unpack(f2_add(a01, a23), u0, u1);
        l_run += u0 + u1;
        // The previous product of this half is complete (its commit preceded this S's).
        if (__any_sync(0xffffffffu, need_rescale)) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            tmem_ld32(t_o + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(t_o + c * 32, o);
          }
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->p_full[s]);
    }
    // Epilogue: normalised fp32 partial and its log2-sum-exp; a half without a key tile, or a row
    // that takes no part, writes the log2-sum-exp -inf only.
    const bool any = n_kv > j0;  // warpgroup-uniform
    const bool seen = ok && any && me.on && !(l_run == 0.f);  // a NaN sum stays one
    const int tile = tile0 + (kKeyPair ? 0 : s);
    const int bl = row / a.group;
    const int b = tile * a.seqs_per_tile + bl;
    const bool stored = bl < a.seqs_per_tile && b < a.batch;
    const int h = kvh * a.group + (row - bl * a.group);
    if (stored && IFA4_DBG_CHECK(a.status, part < a.parts && h < a.n_heads))
      a.ws_lse[(static_cast<long long>(part) * a.batch + b) * a.n_heads + h] =
          seen ? m_run + __log2f(l_run) : -INFINITY;
    if (any && ok && mbar_wait_warp(&bars->o_full[s], 0, ab)) {
      tc_fence_after();
      const float inv_l = seen ? 1.f / l_run : 0.f;
      if (__any_sync(0xffffffffu, stored)) {
        // each lane writes its own row, a 32-byte sector at a time
        float* dst = a.ws_o + ((static_cast<long long>(part) * a.batch + b) * a.n_heads + h) * 128;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(t_o + c * 32, o);
          tmem_wait_ld();
          if (stored && IFA4_DBG_CHECK(a.status, part < a.parts && h < a.n_heads)) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              float f[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(o[8 * v + i]) * inv_l;
              store_sector(dst + c * 32 + 8 * v, f, a.ws_sectors);
            }
          }
          __syncwarp();
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tbase, kTmemCols);
  }
}

// Merge of a row's partials (a.parts of the prefix, a.own_parts of its own keys): weights
// 2^(lse_i - max lse).  kWarps warps share a row's partials, eight in flight each; lanes own 4 of the
// 128 dims, and the warps' sums meet in shared memory.  With four in flight, weights first, one warp
// walking all partials of a row took 20 us for 75 of them (33 sequences x 12 heads) and four 5.8 us;
// with 10 of them (128 x 32 rows) one warp took 6.4 us and four 8.2 us; eight in one pass save 1 to
// 2 us of the whole call (3 sequences behind 32k: 21.4 -> 19.9 us).
constexpr int kCombineThreads = 128;
template <int kWarps>
__global__ void __launch_bounds__(kCombineThreads)
    shared_prefix_combine_kernel(const __grid_constant__ SharedPrefixKernelArgs a) {
  __shared__ __align__(16) float4 sums[kCombineThreads / 32][32];
  __shared__ float weights[kCombineThreads / 32], maxima[kCombineThreads / 32];
  const int warp = (threadIdx.x >> 5) % kWarps, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * (kCombineThreads / 32 / kWarps) +
                        (threadIdx.x >> 5) / kWarps;
  const long long rows = static_cast<long long>(a.batch) * a.n_heads;
  if (row >= rows) return;  // only with one warp per row
  const int b = static_cast<int>(row / a.n_heads);
  const int h = static_cast<int>(row - static_cast<long long>(b) * a.n_heads);
  const int n = a.parts + a.own_parts;
  wait_previous_kernel();  // both kernels' partials (the own keys' ends after the prefix's)
  // Partial i: the prefix's first, then the own keys'.  A warp takes kDepth at a time: sums and
  // outputs are fetched together (an output without weight may never have been written: it is not
  // used), then the running maximum and the sums take them in.
  constexpr int kDepth = 8;
  auto larger = [](float x, float y) { return y > x || y != y ? y : x; };  // a NaN wins
  float m = -INFINITY, wsum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto rescale = [&](float to) {  // to: the new maximum, not -inf
    const float f = m == -INFINITY ? 0.f : fast_exp2(m - to);
    m = to;
    wsum *= f;
    acc.x *= f;
    acc.y *= f;
    acc.z *= f;
    acc.w *= f;
  };
#pragma unroll 1
  for (int i0 = warp * kDepth; i0 < n; i0 += kWarps * kDepth) {
    float l[kDepth];
    float4 o[kDepth];
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      const int i = min(i0 + k, n - 1);
      const bool of_prefix = i < a.parts;
      const long long own = row * a.own_parts + (i - a.parts);
      l[k] = of_prefix ? a.ws_lse[i * rows + row] : a.own_lse[own];
      o[k] = reinterpret_cast<const float4*>(of_prefix ? a.ws_o + (i * rows + row) * 128
                                                       : a.own_o + own * 128)[lane];
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      if (i0 + k >= n) l[k] = -INFINITY;
      mn = larger(mn, l[k]);
    }
    if (mn == -INFINITY) continue;
    rescale(mn);
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      const float wt = fast_exp2(l[k] - m);
      wsum += wt;
      if (wt != 0.f) {
        acc.x += wt * o[k].x;
        acc.y += wt * o[k].y;
        acc.z += wt * o[k].z;
        acc.w += wt * o[k].w;
      }
    }
  }
  if (kWarps > 1) {
    sums[warp][lane] = acc;
    if (lane == 0) {
      weights[warp] = wsum;
      maxima[warp] = m;
    }
    __syncthreads();
    if (warp != 0) return;
    float mn = m;
#pragma unroll
    for (int k = 1; k < kWarps; ++k) mn = larger(mn, maxima[k]);
    if (mn != -INFINITY) {
      rescale(mn);
#pragma unroll
      for (int k = 1; k < kWarps; ++k) {
        const float f = maxima[k] == -INFINITY ? 0.f : fast_exp2(maxima[k] - m);
        const float4 o = sums[k][lane];
        acc.x += f * o.x;
        acc.y += f * o.y;
        acc.z += f * o.z;
        acc.w += f * o.w;
        wsum += f * weights[k];
      }
    }
  }
  const float inv = wsum > 0.f ? 1.f / wsum : (wsum == 0.f ? 0.f : wsum);  // NaN stays
  uint2 packed;
  packed.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  packed.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(a.out + b * a.out_st + h * a.out_sh + lane * 4) = packed;
  if (lane == 0 && a.lse != nullptr)
    a.lse[h * a.lse_sh + b * a.lse_st] =
        wsum == 0.f ? -INFINITY : (m + __log2f(wsum)) * 0.6931471805599453f;
}

}  // namespace prefix

cudaError_t launch_shared_prefix_sm100(const SharedPrefixKernelArgs& args, const CUtensorMap& tm_q,
                                       const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                                       cudaStream_t stream) {
  static std::atomic<bool> attr_rows[64], attr_keys[64];
  cudaError_t e = set_smem_limit_once(prefix::shared_prefix_kernel<false>,
                                      prefix::Layout<false>::kAlloc, attr_rows);
  if (e == cudaSuccess)
    e = set_smem_limit_once(prefix::shared_prefix_kernel<true>, prefix::Layout<true>::kAlloc,
                            attr_keys);
  if (e != cudaSuccess) return e;
  const int tiles = (args.batch + args.seqs_per_tile - 1) / args.seqs_per_tile;
  const dim3 grid(args.key_pair ? tiles : (tiles + 1) / 2, args.kv_heads, args.splits);
  if (args.key_pair)
    prefix::shared_prefix_kernel<true>
        <<<grid, prefix::kThreads, prefix::Layout<true>::kAlloc, stream>>>(args, tm_q, tm_k, tm_v);
  else
    prefix::shared_prefix_kernel<false>
        <<<grid, prefix::kThreads, prefix::Layout<false>::kAlloc, stream>>>(args, tm_q, tm_k, tm_v);
  return cudaGetLastError();
}

cudaError_t launch_shared_prefix_combine_sm100(const SharedPrefixKernelArgs& args,
                                               cudaStream_t stream) {
  const long long rows = static_cast<long long>(args.batch) * args.n_heads;
  constexpr int kT = prefix::kCombineThreads;
  static_assert(kT == 128, "four warps");
  if (args.parts + args.own_parts <= 16)
    return launch_early(prefix::shared_prefix_combine_kernel<1>,
                        dim3(static_cast<unsigned>((rows + 3) / 4)), kT, 0, stream, args);
  return launch_early(prefix::shared_prefix_combine_kernel<4>, dim3(static_cast<unsigned>(rows)), kT,
                      0, stream, args);
}

}  // namespace ifa4
