// Norm and rotation of query and key heads, with or without the append to the paged cache, for
// sm_100a.  One pass over the data, fp32 arithmetic, one rounding to bf16:
//   y   = x * rsqrt(mean_i x_i^2 + eps) * w            (per token and head, 128 dims)
//   out = y with the pairs of its first rotary_dim dims turned by pos * inv_freq_i
// where the pairs are (i, i + rotary_dim / 2) or, interleaved, (2i, 2i + 1), and pos is the
// token's position in its sequence (see IFA4QkNormRopeParams).
//
// Angles: the frequency is kept as a 64-bit fraction of a turn per position, F = frac(inv_freq /
// 2 pi) 2^64, so pos * F modulo 2^64 is the exact fraction of a turn (the integer product wraps
// where the angle does) and no position, however far, loses accuracy to range reduction; its top
// 32 bits go to sincospif (error below 2e-7 rad).
//
// Work split: a unit is one token and a part of its heads; one warp per unit, a half-warp per
// head row (16 lanes x 8 dims, 16-byte loads and stores), four row pairs in flight.  The lane's
// angles depend on the token only, so they are computed once per unit and stay in registers.
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

__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                    pack_bf16x2(x[6], x[7]));
}

// Sum over the 16 lanes of a half-warp.
__device__ __forceinline__ float half_sum(float v) {
#pragma unroll
  for (int m = 8; m > 0; m >>= 1) v += __shfl_xor_sync(kFull, v, m);
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

// The lane's part of a rotation: lane l (of 16) holds dims 8l .. 8l + 7.
//   kRotHalf:  with n = rotary_dim / 16, lanes [0, n) hold the first elements of the pairs and
//              lanes [n, 2n) the second ones; out = own * cos + partner * sin with the sign of
//              the sine folded in; other lanes pass through.
//   kRotPairs: both elements of four pairs are the lane's own.
template <int kRot>
struct Rotation {
  static constexpr int kPairs = kRot == kRotHalf ? 8 : (kRot == kRotPairs ? 4 : 1);
  unsigned long long f[kPairs];
  float c[kPairs], s[kPairs];
  int partner;
  bool turned;   // the lane holds rotated dims
  bool first;    // ... first elements (kRotHalf)

  __device__ __forceinline__ void init(const void* inv_freq, int f32, int rotary_dim, int l) {
    if (kRot == kRotNone) return;
    const int n = kRot == kRotHalf ? rotary_dim / 16 : rotary_dim / 8;
    first = l < n;
    turned = kRot == kRotHalf ? l < 2 * n : l < n;
    partner = kRot == kRotHalf && turned ? (first ? l + n : l - n) : l;
    const int i0 = kRot == kRotHalf ? 8 * (first ? l : l - n) : 4 * l;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) f[i] = turned ? turn_fraction(inv_freq, f32, i0 + i) : 0ull;
  }

  // dir = 1: forward; -1: the transposed rotation (gradients).
  __device__ __forceinline__ void at(long long pos, float dir) {
    if (kRot == kRotNone) return;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      c[i] = 1.f;
      s[i] = 0.f;
    }
    if (turned) {
      const float sign = kRot == kRotHalf && first ? -dir : dir;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        angle_cos_sin(f[i], pos, c[i], s[i]);
        s[i] *= sign;
      }
    }
  }

  // Whole warp.
  __device__ __forceinline__ void apply(float (&y)[8]) const {
    if (kRot == kRotHalf) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = __shfl_sync(kFull, y[i], partner, 16);
      if (turned) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * c[i] + p[i] * s[i];
      }
    } else if (kRot == kRotPairs) {
      if (turned) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = y[2 * i], b = y[2 * i + 1];
          y[2 * i] = a * c[i] - b * s[i];
          y[2 * i + 1] = b * c[i] + a * s[i];
        }
      }
    }
  }
};

// Weight vectors of q and k as fp32 in shared memory (ones when absent).
__device__ __forceinline__ float load_weight(const void* w, int f32, int i) {
  if (w == nullptr) return 1.f;
  return f32 ? __ldg(static_cast<const float*>(w) + i)
             : bf16_bits_to_float(__ldg(static_cast<const uint16_t*>(w) + i));
}

template <int kRot, bool kAppend>
__global__ void __launch_bounds__(kThreads) qkv_rows_kernel(const __grid_constant__
                                                                QkvKernelArgs a) {
  __shared__ __align__(16) float ws[2][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int l = lane & 15, hw = lane >> 4;
  if (a.normalize) {
    ws[0][threadIdx.x] = load_weight(a.q_weight, a.weight_f32, threadIdx.x);
    ws[1][threadIdx.x] = load_weight(a.k_weight, a.weight_f32, threadIdx.x);
  }
  Rotation<kRot> rot;
  rot.init(a.inv_freq, a.inv_freq_f32, a.rotary_dim, l);
  __syncthreads();

  const int rows = a.n_heads + a.kv_heads + (kAppend ? a.kv_heads : 0);
  const long long step = static_cast<long long>(gridDim.x) * kWarps;
  for (long long u = static_cast<long long>(blockIdx.x) * kWarps + warp; u < a.units; u += step) {
    const long long t = a.parts == 1 ? u : u / a.parts;
    const int r0 = static_cast<int>(u - t * a.parts) * a.rows_per_part;
    const int r1 = min(rows, r0 + a.rows_per_part);
    auto source = [&](int r) -> const uint16_t* {
      if (r < a.n_heads) return a.q + t * a.q_st + r * a.q_sh;
      r -= a.n_heads;
      if (!kAppend || r < a.kv_heads) return a.k + t * a.k_st + r * a.k_sh;
      return a.v + t * a.v_st + (r - a.kv_heads) * a.v_sh;
    };
    uint4 x[4];
    auto load4 = [&](int r) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ri = r + 2 * i + hw;
        x[i] = ri < r1 ? ldg_v4(source(ri) + 8 * l) : make_uint4(0u, 0u, 0u, 0u);
      }
    };
    load4(r0);
    const Where w = locate(a.cu_q, a.cu_k, a.batch, t, lane);
    rot.at(w.pos, 1.f);
    long long k_slot = -1, v_slot = -1;  // element offset of the token's slot in the caches
    if (kAppend && w.inside && w.pos >= 0 && (w.pos >> a.page_shift) < a.table_width) {
      const int page = __ldg(a.block_table + static_cast<long long>(w.b) * a.bt_stride +
                             (w.pos >> a.page_shift));
      if (page >= 0 && page < a.num_pages) {
        const long long in_page = w.pos & ((1ll << a.page_shift) - 1);
        k_slot = page * a.kc_sp + in_page * a.kc_st;
        v_slot = page * a.vc_sp + in_page * a.vc_st;
      }
    }
    for (int r = r0; r < r1; r += 8) {
      if (r > r0) load4(r);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ri = r + 2 * i + hw;
        const bool is_q = ri < a.n_heads;
        const bool is_v = kAppend && ri >= a.n_heads + a.kv_heads;
        float y[8];
        unpack8(x[i], y);
        if (a.normalize) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss += y[e] * y[e];
          const float rn = rsqrtf(half_sum(ss) * (1.f / 128.f) + a.eps);
          const float4* wv = reinterpret_cast<const float4*>(ws[is_q ? 0 : 1] + 8 * l);
          const float4 wa = wv[0], wb = wv[1];
          const float wf[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] *= rn * wf[e];
        }
        rot.apply(y);
        uint4 out = is_v ? x[i] : pack8(y);
        uint16_t* dst = nullptr;
        if (ri < r1) {
          if (is_q) {
            dst = a.q_out + t * a.qo_st + ri * a.qo_sh;
          } else if (!kAppend) {
            dst = a.k_out + t * a.ko_st + (ri - a.n_heads) * a.ko_sh;
          } else if (is_v) {
            dst = v_slot >= 0 ? a.v_cache + v_slot + (ri - a.n_heads - a.kv_heads) * a.vc_sh : nullptr;
          } else {
            dst = k_slot >= 0 ? a.k_cache + k_slot + (ri - a.n_heads) * a.kc_sh : nullptr;
          }
          if (!w.inside) {  // behind the last sequence: zeros, or left as it was
            out = make_uint4(0u, 0u, 0u, 0u);
            if (!a.zero_padding) dst = nullptr;
          }
        }
        if (dst != nullptr) *reinterpret_cast<uint4*>(dst + 8 * l) = out;
      }
    }
  }
}

// Gradients.  With g = R^T dout, xhat = x * r, r = rsqrt(mean x^2 + eps):
//   dw = sum over tokens and heads of g * xhat
//   dx = r * (g w - xhat * mean(g w xhat)) = r * g w - x * r^3 * mean(g w x)
// r is recomputed from x (nothing is saved by the forward).  Each half-warp keeps the sums of dw
// of its rows in registers; a block adds its half-warps in a fixed order and writes one partial
// per weight vector, and qkv_weight_grad_kernel adds the blocks' partials, again in a fixed
// order: no atomics, the same result every time.
template <int kRot>
__global__ void __launch_bounds__(kThreads) qkv_backward_kernel(const __grid_constant__
                                                                    QkvBackwardKernelArgs a) {
  __shared__ __align__(16) float ws[2][128];
  __shared__ float part[2][2 * kWarps][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int l = lane & 15, hw = lane >> 4;
  ws[0][threadIdx.x] = load_weight(a.q_weight, a.weight_f32, threadIdx.x);
  ws[1][threadIdx.x] = load_weight(a.k_weight, a.weight_f32, threadIdx.x);
  Rotation<kRot> rot;
  rot.init(a.inv_freq, a.inv_freq_f32, a.rotary_dim, l);
  __syncthreads();
  float acc[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[0][e] = acc[1][e] = 0.f;

  const long long step = static_cast<long long>(gridDim.x) * kWarps;
  for (long long u = static_cast<long long>(blockIdx.x) * kWarps + warp; u < a.units; u += step) {
    const long long t = a.parts == 1 ? u : u / a.parts;
    const int part_i = static_cast<int>(u - t * a.parts);
    const Where w = locate(a.cu_q, a.cu_k, a.batch, t, lane);
    rot.at(w.pos, -1.f);
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const int heads = kind == 0 ? a.n_heads : a.kv_heads;
      const int per = kind == 0 ? a.q_per_part : a.k_per_part;
      const int r0 = part_i * per, r1 = min(heads, r0 + per);
      const uint16_t* xb = kind == 0 ? a.q + t * a.q_st : a.k + t * a.k_st;
      const uint16_t* gb = kind == 0 ? a.dq_out + t * a.dqo_st : a.dk_out + t * a.dko_st;
      uint16_t* ob = kind == 0 ? a.dq + t * a.dq_st : a.dk + t * a.dk_st;
      const long long x_sh = kind == 0 ? a.q_sh : a.k_sh, g_sh = kind == 0 ? a.dqo_sh : a.dko_sh;
      const long long o_sh = kind == 0 ? a.dq_sh : a.dk_sh;
      const float4* wv = reinterpret_cast<const float4*>(ws[kind] + 8 * l);
      const float4 wa = wv[0], wb = wv[1];
      const float wf[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
      for (int r = r0; r < r1; r += 4) {
        uint4 xr[2], gr[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int ri = r + 2 * i + hw;
          const bool on = ri < r1 && w.inside;
          xr[i] = on ? ldg_v4(xb + ri * x_sh + 8 * l) : make_uint4(0u, 0u, 0u, 0u);
          gr[i] = on ? ldg_v4(gb + ri * g_sh + 8 * l) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int ri = r + 2 * i + hw;
          const bool on = ri < r1 && w.inside;  // a row that is none has r = rsqrt(eps), maybe inf
          float x[8], g[8];
          unpack8(xr[i], x);
          unpack8(gr[i], g);
          rot.apply(g);
          if (a.normalize) {
            float ss = 0.f, dot = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              ss += x[e] * x[e];
              dot += g[e] * wf[e] * x[e];
            }
            ss = half_sum(ss);
            dot = half_sum(dot);
            const float rn = rsqrtf(ss * (1.f / 128.f) + a.eps);
            const float back = dot * (1.f / 128.f) * rn * rn;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if (on) acc[kind][e] += g[e] * (x[e] * rn);
              g[e] = rn * (g[e] * wf[e] - x[e] * back);
            }
          }
          if (ri < r1)
            *reinterpret_cast<uint4*>(ob + ri * o_sh + 8 * l) =
                on ? pack8(g) : make_uint4(0u, 0u, 0u, 0u);
        }
      }
    }
  }
  if (a.partial == nullptr) return;
#pragma unroll
  for (int kind = 0; kind < 2; ++kind)
#pragma unroll
    for (int e = 0; e < 8; ++e) part[kind][2 * warp + hw][8 * l + e] = acc[kind][e];
  __syncthreads();
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * kWarps; ++i) s += part[kind][i][threadIdx.x];
    a.partial[(static_cast<long long>(blockIdx.x) * 2 + kind) * 128 + threadIdx.x] = s;
  }
}

// Sum of the blocks' partials: block c adds columns 32 c .. 32 c + 31 of the 256 (q, then k).
__global__ void __launch_bounds__(1024) qkv_weight_grad_kernel(const float* partial, int blocks,
                                                               void* dq_weight, void* dk_weight,
                                                               int f32) {
  __shared__ float s[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), lane_row = threadIdx.x >> 5;
  float acc = 0.f;
  for (int i = lane_row; i < blocks; i += 32) acc += partial[static_cast<long long>(i) * 256 + col];
  s[lane_row][threadIdx.x & 31] = acc;
  __syncthreads();
  if (lane_row == 0) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) sum += s[i][threadIdx.x];
    void* dst = col < 128 ? dq_weight : dk_weight;
    if (dst == nullptr) return;
    if (f32) {
      static_cast<float*>(dst)[col & 127] = sum;
    } else {
      __nv_bfloat16 v = __float2bfloat16_rn(sum);
      static_cast<uint16_t*>(dst)[col & 127] = *reinterpret_cast<uint16_t*>(&v);
    }
  }
}

}  // namespace qkv

cudaError_t launch_qkv_rows_sm100(const QkvKernelArgs& args, int sms, cudaStream_t stream) {
  const long long want = (args.units + qkv::kWarps - 1) / qkv::kWarps;
  const long long cap = static_cast<long long>(sms) * 16;
  const unsigned grid = static_cast<unsigned>(want < cap ? want : cap);
  const int rot = args.rotary_dim == 0 ? qkv::kRotNone
                                       : (args.interleaved ? qkv::kRotPairs : qkv::kRotHalf);
#define IFA4_QKV(R, A)                                                     \
  if (rot == R && (args.k_cache != nullptr) == A) {                        \
    qkv::qkv_rows_kernel<R, A><<<grid, qkv::kThreads, 0, stream>>>(args);  \
    return cudaGetLastError();                                             \
  }
  IFA4_QKV(qkv::kRotNone, false)
  IFA4_QKV(qkv::kRotNone, true)
  IFA4_QKV(qkv::kRotHalf, false)
  IFA4_QKV(qkv::kRotHalf, true)
  IFA4_QKV(qkv::kRotPairs, false)
  IFA4_QKV(qkv::kRotPairs, true)
#undef IFA4_QKV
  return cudaErrorInvalidValue;
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
  qkv::qkv_weight_grad_kernel<<<8, 1024, 0, stream>>>(args.partial, blocks, args.dq_weight,
                                                      args.dk_weight, args.weight_f32);
  return cudaGetLastError();
}

}  // namespace ifa4
