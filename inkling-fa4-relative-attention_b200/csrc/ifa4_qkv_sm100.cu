// Norm and rotation of query and key heads, with or without the append to the paged cache, for
// sm_100a.  One pass over the data, fp32 arithmetic, one rounding to bf16:
//   y   = x * rsqrt(mean_i x_i^2 + eps) * w            (per token and head, 128 dims)
//   out = y with the pairs of its first rotary_dim dims turned by pos * inv_freq_i
// where the pairs are (i, i + rotary_dim / 2) or, interleaved, (2i, 2i + 1), and pos is the
// token's position in its sequence (see IFA4QkNormRopeParams).
//
// Angles: the frequency is kept as a 64-bit fraction of a turn per position, F = frac(inv_freq /
// 2 pi) 2^64, so pos * F modulo 2^64 is the fraction of a turn (the integer product wraps where the
// angle does) and a far position loses nothing to range reduction.  What F itself is off by, the
// rounding of inv_freq / 2 pi in 64 bits, grows with the position as it does in pos * inv_freq: below
// 4e-7 rad at position 2^31 and one radian per position.  The top 32 bits go to sincospif (error below
// 2e-7 rad).
//
// Work split: a unit is one token and a part of its heads; one warp per unit, eight lanes per head
// row (16 dims each, so four rows run at once and a row's sum takes three shuffles), loaded and
// stored in 16-byte pieces.  A lane's dims are chosen so that both elements of its eight pairs are
// its own (8l.. and rotary_dim / 2 + 8l.. for the two halves, 8l.. and 64 + 8l.. interleaved) and so
// that eight lanes' 16 bytes are neighbours: whole sectors in every access.  The angles
// depend on the token only: they are computed once per unit (two pairs a lane), handed round
// through shared memory and kept in registers for all rows.
//
// HBM bound in bytes (671 MB at 32k tokens x 40 heads in 118 us, 5.7 TB/s, where the rotation alone
// runs at 6.1 and a device copy at 6.55), held back by the work per row: 20 warps per SM keep some
// 40 KB of loads in flight, and a quad takes over 200 instructions and a chain of three shuffles
// and a reciprocal root.  The append writes its rows to pages (402 MB in 75 us, 5.4 TB/s; 5.9 for
// the copies alone; V rows have units of their own, 81 us when they were rows of the same units at
// 122 registers), the backward (1007 MB) takes 184 us, 5.5 TB/s.  Measured and slower at those
// sizes: half a warp per row with the pairs exchanged by shuffles 187 us (backward 293); 16
// neighbouring dims a lane, whose accesses cover half sectors, for interleaved pairs 129 instead of
// 105 (30011 tokens); equal runs of quads per warp over token borders 130; whole tokens in turn with
// an evenly cut rest 157; one loop per kind of row (spills) 174; units of one kind, all q first,
// 121-125; the next token streamed by cp.async into shared memory, 8 warps per SM, 126 (append
// 114); backward warps that do q and k rows, with two sets of sums, 194.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ifa4_internal.h"
#include "ifa4_ptx.cuh"

namespace ifa4 {
namespace qkv {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr unsigned kFull = 0xffffffffu;
static_assert(kWarps == kQkvBackwardWarps, "unit planning in the C ABI layer");

enum { kRotNone = 0, kRotHalf = 1, kRotPairs = 2 };

// Plain (coherent) 16-byte load: in-place calls write the rows they read.
__device__ __forceinline__ uint4 ldg_v4(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p)
               : "memory");
  return r;
}

// Eight bf16 <-> eight fp32.  (The rotation in packed fp32 pairs, two values an instruction, was
// slower, 128 us instead of 118 at 32k tokens x 40 heads: it needs the sines' negatives as well.)
__device__ __forceinline__ void unpack8(const uint4& v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint4 pack8(const float* x) {
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                    pack_bf16x2(x[6], x[7]));
}

// Sum over the eight lanes of a row.
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int m = 4; m > 0; m >>= 1) v += __shfl_xor_sync(kFull, v, m);
  return v;
}

struct Where {
  int b;          // sequence
  long long pos;  // position in it
  bool inside;    // false: the row lies behind the last sequence
};

// Sequence and position of token t (whole warp; every lane gets the result).  The largest b with
// cu_q[b] <= t is found 32 candidates at a time.
__device__ __forceinline__ Where locate(const int32_t* cu_q, const int32_t* cu_k, int batch,
                                        long long t, int lane) {
  Where w;
  w.b = 0;
  w.pos = t;
  w.inside = true;
  if (cu_q == nullptr) return w;
  int lo = 0, n = batch;
  if (t < batch && __ldg(cu_q + t) <= t && t < __ldg(cu_q + t + 1)) {
    lo = static_cast<int>(t);  // one token a sequence up to here (decode): no search
    n = 1;
  }
  while (n > 1) {
    const int step = (n + 31) >> 5;
    const int i = lane * step;
    const bool le = i < n && __ldg(cu_q + lo + i) <= t;
    const int c = __popc(__ballot_sync(kFull, le));
    const int skip = c > 0 ? (c - 1) * step : 0;
    lo += skip;
    n = min(step, n - skip);
  }
  const int q0 = __ldg(cu_q + lo), q1 = __ldg(cu_q + lo + 1);
  w.b = lo;
  w.pos = t - q0;
  w.inside = t >= q0 && t < q1;
  if (cu_k != nullptr)
    w.pos += static_cast<long long>(__ldg(cu_k + lo + 1) - __ldg(cu_k + lo)) - (q1 - q0);
  return w;
}

// frac(inv_freq / 2 pi) * 2^64
__device__ __forceinline__ unsigned long long turn_fraction(const void* inv_freq, int f32, int i) {
  const double f = f32 ? static_cast<double>(__ldg(static_cast<const float*>(inv_freq) + i))
                       : __ldg(static_cast<const double*>(inv_freq) + i);
  double turns = f * 0.15915494309189533577;  // 1 / (2 pi)
  turns -= floor(turns);
  return __double2ull_rz(turns * 18446744073709551616.0);
}

__device__ __forceinline__ void angle_cos_sin(unsigned long long f, long long pos, float& c,
                                              float& s) {
  const unsigned long long turn = static_cast<unsigned long long>(pos) * f;
  const int hi = static_cast<int>(turn >> 32);  // signed: [-1/2, 1/2) turn
  sincospif(static_cast<float>(hi) * (1.0f / 2147483648.0f), &s, &c);
}

// The lane's part of a rotation.  Lane l (of 8) of a row holds 16 dims: 8 from a_off on and 8 from
// b_off on, as x[0..7] and x[8..15].
//   kRotHalf:  lanes below n = rotary_dim / 16 hold both halves of the pairs 8l .. 8l + 7; the
//              others share the dims behind rotary_dim, which pass through.
//   kRotPairs: the pairs 4l .. 4l + 3 and 32 + 4l .. 32 + 4l + 3, turned where their dims lie
//              below rotary_dim.
template <int kRot>
struct Rotation {
  unsigned long long f[2];  // frequencies of pairs lane and lane + 32 (the ones this lane computes)
  float c[8], s[8];         // cosines and sines of the lane's own pairs
  int a_off, b_off;
  bool a_turned, b_turned;

  __device__ __forceinline__ void init(const void* inv_freq, int f32, int rotary_dim, int lane) {
    const int l = lane & 7;
    a_off = 8 * l;
    b_off = 64 + 8 * l;
    a_turned = a_off < rotary_dim;
    b_turned = b_off < rotary_dim;
    if (kRot == kRotHalf) {
      const int n = rotary_dim / 16;
      a_turned = b_turned = l < n;
      a_off = a_turned ? 8 * l : rotary_dim + 8 * (l - n);
      b_off = a_turned ? rotary_dim / 2 + 8 * l : rotary_dim + 8 * (8 - n) + 8 * (l - n);
    }
    if (kRot != kRotNone) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        f[i] = lane + 32 * i < rotary_dim / 2 ? turn_fraction(inv_freq, f32, lane + 32 * i) : 0ull;
    }
  }

  // Whole warp; `table` is the warp's own shared memory.
  __device__ __forceinline__ void at(long long pos, int lane, float2* table) {
    if (kRot == kRotNone) return;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float2 cs;
      angle_cos_sin(f[i], pos, cs.x, cs.y);
      table[lane + 32 * i] = cs;
    }
    __syncwarp();
    const int l = lane & 7;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pair = kRot == kRotHalf ? 8 * l + 2 * i : 4 * l + (i < 2 ? 2 * i : 28 + 2 * i);
      const float4 v = *reinterpret_cast<const float4*>(table + pair);  // cos, sin, cos, sin
      c[2 * i] = v.x;
      s[2 * i] = v.y;
      c[2 * i + 1] = v.z;
      s[2 * i + 1] = v.w;
    }
  }

  // Forward, or (kBack) the transposed rotation.
  template <bool kBack>
  __device__ __forceinline__ void apply(float (&x)[16]) const {
    if (kRot == kRotNone || (kRot == kRotHalf && !a_turned)) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (kRot == kRotPairs && (i < 4 ? !a_turned : !b_turned)) continue;
      float& a = kRot == kRotHalf ? x[i] : x[2 * i];
      float& b = kRot == kRotHalf ? x[8 + i] : x[2 * i + 1];
      const float si = kBack ? -s[i] : s[i];
      const float ta = a * c[i] - b * si;
      b = b * c[i] + a * si;
      a = ta;
    }
  }
};

// The lane's 16 weights.
__device__ __forceinline__ void lane_weights(const float* w, int a_off, int b_off, float (&o)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(w + (i < 2 ? a_off + 4 * i : b_off + 4 * (i - 2)));
    o[4 * i] = v.x;
    o[4 * i + 1] = v.y;
    o[4 * i + 2] = v.z;
    o[4 * i + 3] = v.w;
  }
}

// Weight vectors of q and k as fp32 in shared memory (ones when absent).
__device__ __forceinline__ float load_weight(const void* w, int f32, int i) {
  if (w == nullptr) return 1.f;
  return f32 ? __ldg(static_cast<const float*>(w) + i)
             : bf16_bits_to_float(__ldg(static_cast<const uint16_t*>(w) + i));
}

template <int kRot, bool kAppend>
__global__ void __launch_bounds__(kThreads, 5)
    qkv_rows_kernel(const __grid_constant__ QkvKernelArgs a) {
  __shared__ __align__(16) float ws[2][128];
  __shared__ __align__(16) float2 angles[kWarps][64];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int oct = lane >> 3;
  Rotation<kRot> rot;
  rot.init(a.inv_freq, a.inv_freq_f32, a.rotary_dim, lane);
  if (a.normalize) {
    ws[0][threadIdx.x] = load_weight(a.q_weight, a.weight_f32, threadIdx.x);
    ws[1][threadIdx.x] = load_weight(a.k_weight, a.weight_f32, threadIdx.x);
  }
  __syncthreads();

  const int rows = a.n_heads + a.kv_heads;
  // place of a token's rows in a cache (append); null: none
  auto slot = [&](const Where& w, uint16_t* cache, long long sp, long long st) -> uint16_t* {
    if (!w.inside || w.pos < 0 || (w.pos >> a.page_shift) >= a.table_width) return nullptr;
    const int page = __ldg(a.block_table + static_cast<long long>(w.b) * a.bt_stride +
                           (w.pos >> a.page_shift));
    if (page < 0 || page >= a.num_pages) return nullptr;
    return cache + page * sp + (w.pos & ((1ll << a.page_shift) - 1)) * st;
  };
  const long long step = static_cast<long long>(gridDim.x) * kWarps;
  long long u = static_cast<long long>(blockIdx.x) * kWarps + warp;
  for (; u < a.units; u += step) {
    const long long t = a.parts == 1 ? u : u / a.parts;
    const int r0 = static_cast<int>(u - t * a.parts) * a.rows_per_part;
    const int r1 = min(rows, r0 + a.rows_per_part);
    const uint16_t* const qt = a.q + t * a.q_st;
    const uint16_t* const kt = a.k + t * a.k_st;
    uint4 xa[2], xb[2];  // two steps of four rows in flight
    auto load = [&](int r, uint4& va, uint4& vb) {
      const int ri = r + oct;
      va = vb = make_uint4(0u, 0u, 0u, 0u);
      if (ri < r1) {
        const uint16_t* p = ri < a.n_heads ? qt + ri * a.q_sh : kt + (ri - a.n_heads) * a.k_sh;
        va = ldg_v4(p + rot.a_off);
        vb = ldg_v4(p + rot.b_off);
      }
    };
    load(r0, xa[0], xb[0]);
    load(r0 + 4, xa[1], xb[1]);
    const Where w = locate(a.cu_q, a.cu_k, a.batch, t, lane);
    uint16_t* ko;  // the token's rows of k_out, or its slot in the K cache
    if (kAppend) ko = slot(w, a.k_cache, a.kc_sp, a.kc_st);
    else ko = w.inside || a.zero_padding ? a.k_out + t * a.ko_st : nullptr;
    uint16_t* const qo = w.inside || a.zero_padding ? a.q_out + t * a.qo_st : nullptr;
    const long long ko_sh = kAppend ? a.kc_sh : a.ko_sh;
    rot.at(w.pos, lane, angles[warp]);

    auto finish = [&](int r, uint4 va, uint4 vb) {
      const int ri = r + oct;
      const bool is_q = ri < a.n_heads;
      float x[16];
      unpack8(va, x);
      unpack8(vb, x + 8);
      if (a.normalize) {
        float s0 = x[0] * x[0], s1 = x[1] * x[1];
#pragma unroll
        for (int i = 2; i < 16; i += 2) {
          s0 += x[i] * x[i];
          s1 += x[i + 1] * x[i + 1];
        }
        const float rn = rsqrtf(row_sum(s0 + s1) * (1.f / 128.f) + a.eps);
        float wt[16];
        lane_weights(ws[is_q ? 0 : 1], rot.a_off, rot.b_off, wt);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= wt[i] * rn;
      }
      rot.template apply<false>(x);
      va = pack8(x);
      vb = pack8(x + 8);
      if (!w.inside) va = vb = make_uint4(0u, 0u, 0u, 0u);
      uint16_t* const dst = is_q ? qo : ko;
      const long long off = is_q ? ri * a.qo_sh : (ri - a.n_heads) * ko_sh;
      if (ri < r1 && dst != nullptr) {
        *reinterpret_cast<uint4*>(dst + off + rot.a_off) = va;
        *reinterpret_cast<uint4*>(dst + off + rot.b_off) = vb;
      }
    };
    for (int r = r0; r < r1; r += 8) {
      uint4 va = xa[0], vb = xb[0];
      if (r + 8 < r1) load(r + 8, xa[0], xb[0]);
      finish(r, va, vb);
      if (r + 4 < r1) {
        va = xa[1];
        vb = xb[1];
        if (r + 12 < r1) load(r + 12, xa[1], xb[1]);
        finish(r + 4, va, vb);
      }
    }
  }
  if (kAppend) {
    // V rows are copied: a unit is up to eight rows of a token, 16 lanes a row
    const int hw = lane >> 4, l16 = lane & 15;
    for (u -= a.units; u < a.v_units; u += step) {
      const long long t = a.v_parts == 1 ? u : u / a.v_parts;
      const int r0 = static_cast<int>(u - t * a.v_parts) * 8 + hw;
      const uint16_t* const vt = a.v + t * a.v_st + 8 * l16;
      uint4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r0 + 2 * i < a.kv_heads) x[i] = ldg_v4(vt + (r0 + 2 * i) * a.v_sh);
      const Where w = locate(a.cu_q, a.cu_k, a.batch, t, lane);
      uint16_t* const vo = slot(w, a.v_cache, a.vc_sp, a.vc_st);
      if (vo == nullptr) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r0 + 2 * i < a.kv_heads)
          *reinterpret_cast<uint4*>(vo + (r0 + 2 * i) * a.vc_sh + 8 * l16) = x[i];
    }
  }
}

// Gradients.  With g = R^T dout, xhat = x * r, r = rsqrt(mean x^2 + eps):
//   dw = sum over tokens and heads of g * xhat
//   dx = r * (g w - xhat * mean(g w xhat)) = r * g w - x * r^3 * mean(g w x)
// r is recomputed from x (nothing is saved by the forward).  A block works on q rows or on k rows
// only (the blocks are shared out by the work of the two), so a lane keeps one set of 16 sums of dw
// in registers; a block adds its lanes in a fixed order and writes one partial, and
// qkv_weight_grad_kernel adds the blocks' partials, again in a fixed order: no atomics, the same
// result every time.
template <int kRot>
__global__ void __launch_bounds__(kThreads, kQkvBackwardBlocksPerSm)
    qkv_backward_kernel(const __grid_constant__ QkvBackwardKernelArgs a) {
  __shared__ __align__(16) float ws[128];
  __shared__ __align__(16) float2 angles[kWarps][64];
  __shared__ __align__(16) float part[4 * kWarps][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int oct = lane >> 3;
  const bool is_q = blockIdx.x < a.q_blocks;
  const int block = is_q ? blockIdx.x : blockIdx.x - a.q_blocks;
  const int blocks = is_q ? a.q_blocks : gridDim.x - a.q_blocks;
  Rotation<kRot> rot;
  rot.init(a.inv_freq, a.inv_freq_f32, a.rotary_dim, lane);
  ws[threadIdx.x] = load_weight(is_q ? a.q_weight : a.k_weight, a.weight_f32, threadIdx.x);
  __syncthreads();
  const int heads = is_q ? a.n_heads : a.kv_heads;
  const int quads = (heads + 3) / 4;
  const int parts = is_q ? a.q_parts : a.k_parts;
  const uint16_t* const xb = is_q ? a.q : a.k;
  const uint16_t* const gb = is_q ? a.dq_out : a.dk_out;
  uint16_t* const ob = is_q ? a.dq : a.dk;
  const long long x_st = is_q ? a.q_st : a.k_st, x_sh = is_q ? a.q_sh : a.k_sh;
  const long long g_st = is_q ? a.dqo_st : a.dko_st, g_sh = is_q ? a.dqo_sh : a.dko_sh;
  const long long o_st = is_q ? a.dq_st : a.dk_st, o_sh = is_q ? a.dq_sh : a.dk_sh;
  float acc[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;

  const long long units = a.total_q * parts;
  const long long step = static_cast<long long>(blocks) * kWarps;
  for (long long u = static_cast<long long>(block) * kWarps + warp; u < units; u += step) {
    const long long t = parts == 1 ? u : u / parts;
    const int j0 = static_cast<int>(u - t * parts) * a.unit_quads;
    const int r1 = min(heads, 4 * min(j0 + a.unit_quads, quads));
    int ri = 4 * j0 + oct;
    const uint16_t* x_p = xb + t * x_st + ri * x_sh;
    const uint16_t* g_p = gb + t * g_st + ri * g_sh;
    uint16_t* o_p = ob + t * o_st + ri * o_sh;
    uint4 raw[4];  // x, dout of the next four rows
    auto load = [&](int row) {
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (row < r1) {
        raw[0] = ldg_v4(x_p + rot.a_off);
        raw[1] = ldg_v4(x_p + rot.b_off);
        raw[2] = ldg_v4(g_p + rot.a_off);
        raw[3] = ldg_v4(g_p + rot.b_off);
      }
      x_p += 4 * x_sh;
      g_p += 4 * g_sh;
    };
    load(ri);
    const Where w = locate(a.cu_q, a.cu_k, a.batch, t, lane);
    rot.at(w.pos, lane, angles[warp]);
    for (int r = 4 * j0; r < r1; r += 4, ri += 4) {
      const bool on = ri < r1 && w.inside;  // a row that is none has r = rsqrt(eps), maybe inf
      float x[16], g[16];
      unpack8(raw[0], x);
      unpack8(raw[1], x + 8);
      unpack8(raw[2], g);
      unpack8(raw[3], g + 8);
      if (r + 4 < r1) load(ri + 4);
      rot.template apply<true>(g);
      if (a.normalize) {
        float wt[16];
        lane_weights(ws, rot.a_off, rot.b_off, wt);
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          ss += x[i] * x[i];
          dot += g[i] * wt[i] * x[i];
        }
        const float rn = rsqrtf(row_sum(ss) * (1.f / 128.f) + a.eps);
        const float back = row_sum(dot) * (1.f / 128.f) * rn * rn;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (on) acc[i] += g[i] * (x[i] * rn);
          g[i] = rn * (g[i] * wt[i] - x[i] * back);
        }
      }
      if (ri < r1) {
        const uint4 z = make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4*>(o_p + rot.a_off) = on ? pack8(g) : z;
        *reinterpret_cast<uint4*>(o_p + rot.b_off) = on ? pack8(g + 8) : z;
      }
      o_p += 4 * o_sh;
    }
  }
  if (a.partial == nullptr) return;
  launch_dependents();  // the sum over blocks
#pragma unroll
  for (int i = 0; i < 16; ++i)
    part[4 * warp + oct][i < 8 ? rot.a_off + i : rot.b_off + i - 8] = acc[i];
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 4 * kWarps; ++i) sum += part[i][threadIdx.x];
  a.partial[static_cast<long long>(blockIdx.x) * 128 + threadIdx.x] = sum;
}

// Sum of the blocks' partials ([q_blocks][128], then those of k): block c adds 32 columns of q
// (c < 4) or of k.
__global__ void __launch_bounds__(1024) qkv_weight_grad_kernel(const float* partial, int q_blocks,
                                                               int blocks, void* dq_weight,
                                                               void* dk_weight, int f32) {
  __shared__ float s[32][33];
  const bool is_q = blockIdx.x < 4;
  const int col = (blockIdx.x & 3) * 32 + (threadIdx.x & 31), lane_row = threadIdx.x >> 5;
  const int first = is_q ? 0 : q_blocks, last = is_q ? q_blocks : blocks;
  wait_previous_kernel();
  float acc = 0.f;
  for (int i = first + lane_row; i < last; i += 32)
    acc += partial[static_cast<long long>(i) * 128 + col];
  s[lane_row][threadIdx.x & 31] = acc;
  __syncthreads();
  if (lane_row == 0) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) sum += s[i][threadIdx.x];
    void* dst = is_q ? dq_weight : dk_weight;
    if (dst == nullptr) return;
    if (f32) {
      static_cast<float*>(dst)[col] = sum;
    } else {
      __nv_bfloat16 v = __float2bfloat16_rn(sum);
      static_cast<uint16_t*>(dst)[col] = *reinterpret_cast<uint16_t*>(&v);
    }
  }
}

}  // namespace qkv

// Blocks of one kernel that are resident on the current device at a time.
template <typename K>
static cudaError_t resident_blocks(K kernel, int sms, std::atomic<int> (&cache)[64], int* out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  int n = cache[dev].load(std::memory_order_acquire);
  if (n == 0) {
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, qkv::kThreads, 0);
    if (e != cudaSuccess) return e;
    if (n < 1) n = 1;
    cache[dev].store(n, std::memory_order_release);
  }
  *out = n * sms;
  return cudaSuccess;
}

template <int kRot, bool kAppend>
static cudaError_t launch_rows(const QkvKernelArgs& args, int sms, cudaStream_t stream) {
  static std::atomic<int> cache[64];
  int cap = 0;
  cudaError_t e = resident_blocks(qkv::qkv_rows_kernel<kRot, kAppend>, sms, cache, &cap);
  if (e != cudaSuccess) return e;
  const long long want = (args.units + args.v_units + qkv::kWarps - 1) / qkv::kWarps;
  const unsigned grid = static_cast<unsigned>(want < cap ? want : cap);
  qkv::qkv_rows_kernel<kRot, kAppend><<<grid, qkv::kThreads, 0, stream>>>(args);
  return cudaGetLastError();
}

cudaError_t launch_qkv_rows_sm100(const QkvKernelArgs& args, int sms, cudaStream_t stream) {
  const bool append = args.k_cache != nullptr;
  if (args.rotary_dim == 0)
    return append ? launch_rows<qkv::kRotNone, true>(args, sms, stream)
                  : launch_rows<qkv::kRotNone, false>(args, sms, stream);
  if (args.interleaved)
    return append ? launch_rows<qkv::kRotPairs, true>(args, sms, stream)
                  : launch_rows<qkv::kRotPairs, false>(args, sms, stream);
  return append ? launch_rows<qkv::kRotHalf, true>(args, sms, stream)
                : launch_rows<qkv::kRotHalf, false>(args, sms, stream);
}

cudaError_t launch_qkv_backward_sm100(const QkvBackwardKernelArgs& args, int blocks,
                                      cudaStream_t stream) {
  const int rot = args.rotary_dim == 0 ? qkv::kRotNone
                                       : (args.interleaved ? qkv::kRotPairs : qkv::kRotHalf);
  if (rot == qkv::kRotNone)
    qkv::qkv_backward_kernel<qkv::kRotNone><<<blocks, qkv::kThreads, 0, stream>>>(args);
  else if (rot == qkv::kRotHalf)
    qkv::qkv_backward_kernel<qkv::kRotHalf><<<blocks, qkv::kThreads, 0, stream>>>(args);
  else
    qkv::qkv_backward_kernel<qkv::kRotPairs><<<blocks, qkv::kThreads, 0, stream>>>(args);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || args.partial == nullptr) return e;
  return launch_early(qkv::qkv_weight_grad_kernel, dim3(8), 1024, 0, stream,
                      const_cast<const float*>(args.partial), args.q_blocks, blocks, args.dq_weight,
                      args.dk_weight, args.weight_f32);
}

}  // namespace ifa4
