// Learned relative position bias by distance buckets for sm_100a, and its gradient.
//   rel[h, d]    = table[bucket(d), h]                               0 <= d < rel_extent
//   grad[b, h]   = sum over tokens t and distances d of bucket b of drel[t, h, d]
// bucket(d) is the last bucket whose start is <= d (ascending starts; bucket 0 also takes what
// lies before its start).
//
// The forward writes one [n_heads, rel_extent] table, which the attention reads with token
// stride 0 (2 us, its launch).  The gradient is one read of drel, HBM bound: 268 MB (32k tokens x 32
// heads x 128) in 43 us, 6.2 TB/s, and 2.15 GB (x 1024) in 297 us, 7.2 TB/s, what a read-only stream
// reaches; the shorter one pays its start and its bucket sums.  A thread owns V neighbouring columns
// of one head and adds its tokens in registers (fp32, eight loads in flight), a block adds its
// token lanes and then its columns by bucket in a fixed order and writes one partial per head and
// bucket; a second kernel adds the blocks' partials in a fixed order (no atomics).  With a single
// token chunk the first kernel writes the result itself.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>

#include "ifa4_internal.h"
#include "ifa4_ptx.cuh"

namespace ifa4 {
namespace bucket {

constexpr int kThreads = 256;

__device__ __forceinline__ void store_as(void* dst, long long i, float v, int f32) {
  if (f32) {
    static_cast<float*>(dst)[i] = v;
  } else {
    __nv_bfloat16 b = __float2bfloat16_rn(v);
    static_cast<uint16_t*>(dst)[i] = *reinterpret_cast<uint16_t*>(&b);
  }
}

__global__ void __launch_bounds__(kThreads) bucket_bias_kernel(const __grid_constant__
                                                                   BucketBiasKernelArgs a) {
  __shared__ int starts[kMaxBuckets];
  for (int i = threadIdx.x; i < a.buckets; i += kThreads) starts[i] = __ldg(a.starts + i);
  __syncthreads();
  const int d = blockIdx.x * kThreads + threadIdx.x;
  const int h = blockIdx.y;
  if (d >= a.rel_extent) return;
  int lo = 0, hi = a.buckets - 1;  // last bucket with starts[b] <= d, bucket 0 if none
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= d) lo = mid; else hi = mid - 1;
  }
  const long long i = lo * a.table_sb + h * a.table_sh;
  const float v = a.table_f32 ? __ldg(static_cast<const float*>(a.table) + i)
                              : bf16_bits_to_float(__ldg(static_cast<const uint16_t*>(a.table) + i));
  __nv_bfloat16 b = __float2bfloat16_rn(v);
  a.rel[h * a.rel_sh + d] = *reinterpret_cast<uint16_t*>(&b);
}

template <int V>
struct Vec;
template <>
struct Vec<8> {
  uint4 v;
  __device__ __forceinline__ void load(const uint16_t* p) { v = ldg_nc_v4(p); }
  __device__ __forceinline__ void add(float (&s)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[2 * i] += __uint_as_float(w[i] << 16);
      s[2 * i + 1] += __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <>
struct Vec<4> {
  uint2 v;
  __device__ __forceinline__ void load(const uint16_t* p) {
    v = __ldg(reinterpret_cast<const uint2*>(p));
  }
  __device__ __forceinline__ void add(float (&s)[4]) const {
    s[0] += __uint_as_float(v.x << 16);
    s[1] += __uint_as_float(v.x & 0xffff0000u);
    s[2] += __uint_as_float(v.y << 16);
    s[3] += __uint_as_float(v.y & 0xffff0000u);
  }
};
template <>
struct Vec<2> {
  uint32_t v;
  __device__ __forceinline__ void load(const uint16_t* p) {
    v = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
  __device__ __forceinline__ void add(float (&s)[2]) const {
    s[0] += __uint_as_float(v << 16);
    s[1] += __uint_as_float(v & 0xffff0000u);
  }
};
template <>
struct Vec<1> {
  uint16_t v;
  __device__ __forceinline__ void load(const uint16_t* p) { v = __ldg(p); }
  __device__ __forceinline__ void add(float (&s)[1]) const { s[0] += bf16_bits_to_float(v); }
};

// Block (x, y): column block x = (head block, column part), token chunk y.  A block covers
// a.heads heads x a.cols columns (columns of one head from a.cols * part on), a.lanes token lanes.
// With a.flat the heads lie one behind the other and a thread's columns may cross from one to the
// next (rel_extent is then not a multiple of V, the columns of a block are).
template <int V>
__global__ void __launch_bounds__(kThreads) bucket_grad_kernel(const __grid_constant__
                                                                   BucketGradKernelArgs a) {
  __shared__ float sums[kThreads * V];      // [lane][head][column]
  __shared__ int starts[kMaxBuckets + 1];
  for (int i = threadIdx.x; i <= a.buckets; i += kThreads)
    starts[i] = i == 0 ? 0 : (i == a.buckets ? a.rel_extent
                                              : min(max(__ldg(a.starts + i), 0), a.rel_extent));
  const int part = blockIdx.x % a.col_parts;
  const int h0 = (blockIdx.x / a.col_parts) * a.heads;
  const int e0 = part * a.cols;
  const int n_cols = min(a.cols, a.rel_extent - e0);
  const int vecs = a.flat ? a.heads * a.cols / V : a.cols / V;  // threads of a head, or of a lane
  const int per_lane = a.flat ? vecs : a.heads * vecs;          // threads of a token lane
  const int lane = threadIdx.x / per_lane;
  const int in_lane = threadIdx.x - lane * per_lane;
  const int hl = a.flat ? 0 : in_lane / vecs;
  const int c = (in_lane - hl * vecs) * V;
  const int c_end = a.flat ? min(a.heads, a.n_heads - h0) * a.rel_extent : n_cols;
  long long tokens = a.total_q;
  if (a.cu_q != nullptr) tokens = min(tokens, static_cast<long long>(max(__ldg(a.cu_q + a.batch), 0)));
  const long long t0 = blockIdx.y * a.chunk;
  const long long t1 = min(tokens, t0 + a.chunk);
  const bool on = lane < a.lanes && h0 + hl < a.n_heads && c < c_end;
  float s[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = 0.f;
  if (on) {
    const long long step = static_cast<long long>(a.lanes) * a.drel_st;
    long long t = t0 + lane;
    const uint16_t* p = a.drel + t * a.drel_st + (h0 + hl) * a.drel_sh + e0 + c;
    for (; t + 7 * a.lanes < t1; t += 8 * a.lanes) {
      Vec<V> x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i].load(p + i * step);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i].add(s);
      p += 8 * step;
    }
    Vec<V> x[7];  // the last tokens, all loads in flight as well
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (t + i * a.lanes < t1) x[i].load(p + i * step);
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (t + i * a.lanes < t1) x[i].add(s);
  }
  if (lane < a.lanes) {
#pragma unroll
    for (int i = 0; i < V; ++i) sums[(lane * a.heads + hl) * a.cols + c + i] = s[i];
  }
  __syncthreads();
  // columns: add the token lanes
  const int width = a.heads * a.cols;
  if (a.lanes > 1) {
    for (int i = threadIdx.x; i < width; i += kThreads) {
      float v = sums[i];
      for (int k = 1; k < a.lanes; ++k) v += sums[k * width + i];
      sums[i] = v;
    }
    __syncthreads();
  }
  launch_dependents();  // the sum over slots
  // buckets: a thread per head and bucket, eight where buckets hold 16 columns and more on average
  const int per = a.rel_extent >= 16 * a.buckets ? 8 : 1;
  const int sub = threadIdx.x & (per - 1);
  const int tasks = a.heads * a.buckets;
  for (int task0 = 0; task0 < tasks; task0 += kThreads / per) {
    const int task = task0 + threadIdx.x / per;
    const int th = task < tasks ? task / a.buckets : 0;
    const int b = task - th * a.buckets;
    float v = 0.f;
    if (task < tasks) {
      const int lo = max(starts[b] - e0, 0), hi = min(starts[b + 1] - e0, n_cols);
      for (int i = lo + sub; i < hi; i += per) v += sums[th * a.cols + i];
    }
    if (per == 8) {
      v += __shfl_xor_sync(0xffffffffu, v, 4);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      v += __shfl_xor_sync(0xffffffffu, v, 1);
    }
    if (sub == 0 && task < tasks && h0 + th < a.n_heads) {
      if (a.slots == 1)
        store_as(a.grad, b * a.grad_sb + (h0 + th) * a.grad_sh, v, a.grad_f32);
      else
        a.partial[((static_cast<long long>(blockIdx.y) * a.col_parts + part) * a.n_heads + h0 + th) *
                      a.buckets + b] = v;
    }
  }
}

// grad[b, h] = sum over slots of partial[slot][h][b]; a block adds 32 neighbouring (h, b).
__global__ void __launch_bounds__(1024) bucket_grad_sum_kernel(const __grid_constant__
                                                                   BucketGradKernelArgs a) {
  __shared__ float s[32][33];
  const int n = a.n_heads * a.buckets;
  const int i = blockIdx.x * 32 + (threadIdx.x & 31), row = threadIdx.x >> 5;
  wait_previous_kernel();
  float acc = 0.f;
  if (i < n)
    for (int k = row; k < a.slots; k += 32) acc += a.partial[static_cast<long long>(k) * n + i];
  s[row][threadIdx.x & 31] = acc;
  __syncthreads();
  if (row == 0 && i < n) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) v += s[k][threadIdx.x];
    store_as(a.grad, (i % a.buckets) * a.grad_sb + (i / a.buckets) * a.grad_sh, v, a.grad_f32);
  }
}

}  // namespace bucket

cudaError_t launch_bucket_bias_sm100(const BucketBiasKernelArgs& args, cudaStream_t stream) {
  const dim3 grid((args.rel_extent + bucket::kThreads - 1) / bucket::kThreads, args.n_heads);
  bucket::bucket_bias_kernel<<<grid, bucket::kThreads, 0, stream>>>(args);
  return cudaGetLastError();
}

// Column blocks and token chunks of the gradient (fills flat, heads, cols, col_parts, lanes, chunk,
// slots of `a` from its sizes).  Returns the columns a thread loads at once: the most the layout
// allows.  Where rel_extent is not a multiple of eight but the heads lie one behind the other, a
// block takes whole heads as one row of columns (32k x 32 x 100: 76 us in pairs of columns,
// 39 us).
int plan_bucket_grad(BucketGradKernelArgs* a, int sms) {
  auto loads = [&](int v) {  // rows of columns in pieces of v
    return reinterpret_cast<uintptr_t>(a->drel) % (2 * v) == 0 && a->drel_st % v == 0;
  };
  int vec = 1, together = 1;  // together: heads whose columns make whole pieces
  a->flat = 0;
  for (int v : {8, 4, 2})
    if (loads(v) && a->drel_sh % v == 0 && a->rel_extent % v == 0) {
      vec = v;
      break;
    }
  if (vec < 8 && loads(8) && a->drel_sh == a->rel_extent &&
      static_cast<long long>(a->n_heads) * a->rel_extent % 8 == 0) {
    while (static_cast<long long>(together) * a->rel_extent % 8 != 0) together *= 2;
    if (together * static_cast<long long>(a->rel_extent) <= bucket::kThreads * 8) {
      a->flat = 1;
      vec = 8;
    }
  }
  if (a->flat) {
    a->cols = a->rel_extent;
    a->col_parts = 1;
    int heads = bucket::kThreads * 8 / a->rel_extent / together * together;
    const int all = (a->n_heads + together - 1) / together * together;
    a->heads = heads < all ? heads : all;
    a->lanes = bucket::kThreads / (a->heads * a->rel_extent / 8);
  } else {
    const int vecs = a->rel_extent / vec;
    const int head_vecs = vecs < bucket::kThreads ? vecs : bucket::kThreads;
    a->cols = head_vecs * vec;
    a->col_parts = (vecs + head_vecs - 1) / head_vecs;
    // heads of a block: the count that leaves the fewest threads without columns, the larger one
    // of equals
    int most_heads = bucket::kThreads / head_vecs;
    if (most_heads > a->n_heads) most_heads = a->n_heads;
    double best = 0;
    for (int heads = most_heads; heads >= 1; --heads) {
      const int lanes = bucket::kThreads / (heads * head_vecs);
      const int blocks = (a->n_heads + heads - 1) / heads;
      const double used = static_cast<double>(a->n_heads) / (blocks * heads) * heads * head_vecs * lanes;
      if (used > best * 1.001) {
        best = used;
        a->heads = heads;
        a->lanes = lanes;
      }
    }
  }
  const long long col_blocks =
      static_cast<long long>((a->n_heads + a->heads - 1) / a->heads) * a->col_parts;
  // one resident wave of blocks (four per SM; 32k tokens x 32 heads x 128: 43 us, 46 us with two
  // waves of half the tokens, 44 us with three blocks), at least 32 tokens per lane (one chunk needs
  // no second kernel)
  long long chunks = 4ll * sms / col_blocks;
  const long long most = (a->total_q + 32ll * a->lanes - 1) / (32ll * a->lanes);
  if (chunks > most) chunks = most;
  if (chunks < 1) chunks = 1;
  if (chunks > 65535) chunks = 65535;
  a->chunk = (a->total_q + chunks - 1) / chunks;
  if (a->chunk < 1) a->chunk = 1;  // no token: one block column writes the zeros
  a->chunks = static_cast<int>((a->total_q + a->chunk - 1) / a->chunk);
  if (a->chunks < 1) a->chunks = 1;
  a->slots = a->chunks * a->col_parts;
  return vec;
}

cudaError_t launch_bucket_grad_sm100(const BucketGradKernelArgs& args, int vec,
                                     cudaStream_t stream) {
  const dim3 grid((args.n_heads + args.heads - 1) / args.heads * args.col_parts, args.chunks);
  if (vec == 8)
    bucket::bucket_grad_kernel<8><<<grid, bucket::kThreads, 0, stream>>>(args);
  else if (vec == 4)
    bucket::bucket_grad_kernel<4><<<grid, bucket::kThreads, 0, stream>>>(args);
  else if (vec == 2)
    bucket::bucket_grad_kernel<2><<<grid, bucket::kThreads, 0, stream>>>(args);
  else
    bucket::bucket_grad_kernel<1><<<grid, bucket::kThreads, 0, stream>>>(args);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || args.slots == 1) return e;
  const int n = args.n_heads * args.buckets;
  return launch_early(bucket::bucket_grad_sum_kernel, dim3((n + 31) / 32), 1024, 0, stream, args);
}

}  // namespace ifa4
