// Internal interface between the C ABI layer (ifa4_capi.cu) and the kernel translation units.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace ifa4 {

constexpr int kHeadDim = 128;

// Raises a kernel's dynamic shared-memory limit on the current device, once per device (the
// limit is a per-device function attribute).  `done` is one flag per device ordinal; it is
// atomic, so host threads launching at the same time do not race on it (two first calls may
// both set the attribute, which is harmless: the value is the same).
template <typename K>
cudaError_t set_smem_limit_once(K kernel, uint32_t bytes, std::atomic<bool> (&done)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!done[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(bytes));
    if (e != cudaSuccess) return e;
    done[dev].store(true, std::memory_order_release);
  }
  return cudaSuccess;
}

// Launch that may start before the previous kernel of the stream has finished, as soon as all of its
// blocks have called launch_dependents() (see ifa4_ptx.cuh) or ended.
template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, int threads, uint32_t smem,
                         cudaStream_t stream, const A&... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Status bits written by kernels that abandoned a bounded wait.
constexpr int kStatusPrefillTimeout = 1;
constexpr int kStatusDecodeTimeout = 2;
constexpr int kStatusBackwardTimeout = 4;
constexpr int kStatusSelfTestTimeout = 8;   // ifa4_selftest_bounded_wait, warp 0
constexpr int kStatusSelfTestOwnTimeout = 16;  // ifa4_selftest_bounded_wait, warp 1 (must not be set)
constexpr int kStatusRelLogitsTimeout = 32;
constexpr int kStatusDebugBounds = 64;   // debug builds only: an index range check failed

// Index range checks of debug builds (compiled with -DIFA4_DEBUG, the library's stand-in for a
// bounds-checking sanitizer): a failed check ORs kStatusDebugBounds into the status word and the
// guarded access is skipped, so a bad index is reported without touching memory out of range.
// In release builds the condition is not evaluated and the access is unconditional.
#ifdef IFA4_DEBUG
__device__ __forceinline__ bool debug_check(int* status, bool ok) {
  if (!ok && status != nullptr) atomicOr(status, kStatusDebugBounds);
  return ok;
}
#define IFA4_DBG_CHECK(status, cond) ::ifa4::debug_check((status), (cond))
#else
#define IFA4_DBG_CHECK(status, cond) true
#endif

struct PrefillKernelArgs {
  const uint16_t* rel;       // bf16 bits
  uint16_t* out;             // bf16 bits
  const int32_t* cu_q;
  const int32_t* cu_k;
  long long rel_st, rel_sh;
  long long out_st, out_sh;
  int batch, n_heads, kv_heads, rel_extent;
  int causal, window_left, align_bottom_right;
  int bias_vec;              // rel 16-byte aligned (base, strides) and rel_extent % 8 == 0:
                             // each row loads its bias with 16-byte vectors
  int pair_heads;            // 1: the CTA's two sub-tiles are two heads at the same rows
                             // 0: the CTA's two sub-tiles are consecutive 128-row blocks
  int q_fastest;             // grid (query slots, head slots, sequences) rather than
                             // (head slots, sequences, query slots)
  float scale_log2;          // softmax_scale * log2(e)
  float* lse;                // optional natural-log LSE, [h * lse_sh + token * lse_st]
  long long lse_sh, lse_st;
  // paged KV cache (kernels instantiated with kPaged): K/V tensor maps are 4-D
  // {128 dims, kv_heads, page_size, num_pages}; tiles load in units of 2^box_shift rows
  const int32_t* block_table;
  long long bt_stride;
  int page_shift, box_shift, num_pages;
  const uint16_t* v;         // V cache base (partial last unit copied with plain loads)
  long long v_st, v_sh, v_sp;
  int* status;
  // output copies on other GPUs: element e of out is also stored at out + out_peer_delta[i] + e
  long long out_peer_delta[7];
  int n_out_peers;
  // KV split (kv_splits > 1): the query tile's KV tiles are cut into kv_splits ranges, one per
  // CTA; each writes its rows' normalised fp32 partial output and log2-sum-exp, and
  // rel_attn_prefill_combine_kernel merges them into out (and lse)
  int kv_splits;
  float* ws_o;               // [kv_splits, total_q, n_heads, 128]
  float* ws_lse;             // [kv_splits, n_heads, total_q], log2 units, -inf: no visible key
  long long total_q;
};

struct PrefillLaunch {
  dim3 grid;
  int smem_bytes;
};

// Prefill tile configurations: the kernel variants differ in where the exponentials of every 16
// score columns are computed: FMA-pipe polynomial, SFU two-at-a-time (f16x2), or SFU fp32.
// tile_config 0 = automatic (2 polynomial columns of 16); 1..5 = 0, 2, 4, 6, 8 polynomial columns of 16; 6 = all f16x2; 7 = 8 of 16 f16x2;
// 8 = 4 polynomial + 8 f16x2.
constexpr int kPrefillDefaultEmu = 2;
constexpr int kPrefillDefaultHalf2 = 0;
constexpr int kPrefillNumTileConfigs = 9;
int prefill_emulated_exp_columns(int tile_config);  // -1 for an unknown id

// Launches the tcgen05 prefill kernel variant of `tile_config`.  Returns a cudaError_t.
// With a paged cache (args.block_table != nullptr) only tile configs 0 to 3 exist.
cudaError_t launch_prefill_sm100(const PrefillKernelArgs& args, const CUtensorMap& tm_q,
                                 const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                                 int q_slots, int tile_config, int max_seqlen_q,
                                 cudaStream_t stream);
// Merge of the kv_splits partials written by a split launch (one warp per token and head).
cudaError_t launch_prefill_combine_sm100(const PrefillKernelArgs& args, cudaStream_t stream);
bool prefill_paged_tile_config_ok(int tile_config);

struct DecodeKernelArgs {
  const uint16_t* q;
  const uint16_t* rel;
  uint16_t* out;
  const int32_t* cu_q;
  const int32_t* cu_k;
  long long q_st, q_sh;
  long long rel_st, rel_sh;
  long long out_st, out_sh;
  int batch, n_heads, kv_heads, rel_extent;
  int causal, window_left, align_bottom_right;
  int group;                 // n_heads / kv_heads
  int heads_per_cta;         // <= 16 query heads of one kv group per CTA
  int num_splits;            // CTAs per (sequence, head block)
  int chunk_len;             // keys per chunk (multiple of 64)
  float scale_log2;
  float* ws_o;               // [batch, n_heads, num_splits, 128] (num_splits > 1)
  float* ws_lse;             // [batch, n_heads, num_splits]      (num_splits > 1)
  float* lse;                // optional natural-log LSE output
  long long lse_sh, lse_st;
  const int32_t* block_table;  // paged KV cache, as in PrefillKernelArgs
  long long bt_stride;
  int page_shift, box_shift, num_pages;
  // shared prefix (0: none): sequences of at least this many keys start at key prefix_len.  With one
  // split the CTA merges the prefix's partials itself (px_*, as SharedPrefixKernelArgs has them);
  // otherwise its own go to shared_prefix_combine_kernel
  int prefix_len;
  const float* px_o;
  const float* px_lse;
  int px_parts;
  int* status;
};

cudaError_t launch_decode_sm100(const DecodeKernelArgs& args, const CUtensorMap& tm_k,
                                const CUtensorMap& tm_v, cudaStream_t stream);

// Prefix part of a decode batch that shares its first prefix_len keys, and the merge with the
// sequences' own keys (decode partials own_o / own_lse).
struct SharedPrefixKernelArgs {
  const uint16_t* rel;
  long long rel_st, rel_sh;
  const int32_t* cu_k;
  int batch, n_heads, kv_heads, rel_extent;
  int group;                 // n_heads / kv_heads
  int seqs_per_tile;         // 128 / group: sequences in a 128-row tile
  int prefix_len, window_left;
  int key_pair;              // one row tile per KV head: halves alternate over key tiles
  int splits;                // key splits (CTAs per row tile pair and KV head)
  int parts;                 // prefix partials per row: splits, or 2 * splits with key_pair
  int bias_vec;              // as in PrefillKernelArgs
  float scale_log2;
  const int32_t* block_table;
  long long bt_stride;
  int page_shift, box_shift, num_pages;
  const uint16_t* v;         // V cache base (the unit in which the prefix ends)
  long long v_st, v_sh, v_sp;
  float* ws_o;               // [parts, batch, n_heads, 128], 16-byte aligned
  int ws_sectors;            // ws_o is 32-byte aligned
  float* ws_lse;             // [parts, batch, n_heads], log2 units, -inf: no visible key
  const float* own_o;        // [batch, n_heads, own_parts, 128]
  const float* own_lse;      // [batch, n_heads, own_parts]
  int own_parts;
  uint16_t* out;
  long long out_st, out_sh;
  float* lse;                // optional natural-log LSE
  long long lse_sh, lse_st;
  int* status;
};

cudaError_t launch_shared_prefix_sm100(const SharedPrefixKernelArgs& args, const CUtensorMap& tm_q,
                                       const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                                       cudaStream_t stream);
cudaError_t launch_shared_prefix_combine_sm100(const SharedPrefixKernelArgs& args,
                                               cudaStream_t stream);

// Norm and rotation of q and k rows; with k_cache set, k and v rows go to the paged caches.
struct QkvKernelArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* q_out;
  uint16_t* k_out;
  uint16_t* k_cache;
  uint16_t* v_cache;
  const void* q_weight;      // [128] bf16 or fp32, null: ones
  const void* k_weight;
  const void* inv_freq;      // [rotary_dim / 2] fp64 or fp32
  const int32_t* cu_q;       // optional (null: one sequence)
  const int32_t* cu_k;       // optional
  const int32_t* block_table;
  long long q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh, ko_st, ko_sh;
  long long kc_sp, kc_st, kc_sh, vc_sp, vc_st, vc_sh;
  long long bt_stride;
  long long units;           // total_q * parts
  int batch, n_heads, kv_heads;
  int rotary_dim, interleaved, normalize, weight_f32, inv_freq_f32, zero_padding;
  long long v_units;         // append: total_q * v_parts units of V rows behind them
  int v_parts;               // ceil(kv_heads / 8)
  int parts, rows_per_part;  // a token's q and k rows are shared by `parts` warps
  int page_shift, table_width, num_pages;
  float eps;
};

struct QkvBackwardKernelArgs {
  const uint16_t* dq_out;
  const uint16_t* dk_out;
  const uint16_t* q;
  const uint16_t* k;
  uint16_t* dq;
  uint16_t* dk;
  const void* q_weight;
  const void* k_weight;
  void* dq_weight;           // optional, like the weights
  void* dk_weight;
  const void* inv_freq;
  const int32_t* cu_q;
  const int32_t* cu_k;
  float* partial;            // [blocks, 128], q's first (null: no weight gradients)
  long long dqo_st, dqo_sh, dko_st, dko_sh, q_st, q_sh, k_st, k_sh, dq_st, dq_sh, dk_st, dk_sh;
  long long total_q;
  int batch, n_heads, kv_heads;
  int rotary_dim, interleaved, normalize, weight_f32, inv_freq_f32;
  int q_blocks;              // the first blocks work on q, the others on k
  int unit_quads;            // most quads (four rows) of a unit
  int q_parts, k_parts;      // units of a token's q, and of its k
  float eps;
};

cudaError_t launch_qkv_rows_sm100(const QkvKernelArgs& args, int sms, cudaStream_t stream);
cudaError_t launch_qkv_backward_sm100(const QkvBackwardKernelArgs& args, int blocks,
                                      cudaStream_t stream);
constexpr int kQkvBackwardWarps = 4;        // warps of a block of the backward kernel
constexpr int kQkvBackwardBlocksPerSm = 4;  // resident ones

// Bias by distance buckets and its gradient.
constexpr int kMaxBuckets = 1024;
struct BucketBiasKernelArgs {
  const void* table;         // table[b * table_sb + h * table_sh], bf16 or fp32
  const int32_t* starts;     // [buckets]
  uint16_t* rel;             // rel[h * rel_sh + d]
  long long table_sb, table_sh, rel_sh;
  int n_heads, rel_extent, buckets, table_f32;
};
struct BucketGradKernelArgs {
  const uint16_t* drel;
  const int32_t* starts;
  const int32_t* cu_q;       // optional: tokens from cu_q[batch] on are not counted
  void* grad;                // grad[b * grad_sb + h * grad_sh], bf16 or fp32
  float* partial;            // [slots, n_heads, buckets]
  long long drel_st, drel_sh, grad_sb, grad_sh;
  long long total_q, chunk;  // tokens, tokens per chunk
  int batch, n_heads, rel_extent, buckets, grad_f32;
  int flat, heads, cols, col_parts, lanes, chunks, slots;  // plan_bucket_grad
};
cudaError_t launch_bucket_bias_sm100(const BucketBiasKernelArgs& args, cudaStream_t stream);
int plan_bucket_grad(BucketGradKernelArgs* a, int sms);
cudaError_t launch_bucket_grad_sm100(const BucketGradKernelArgs& args, int vec,
                                     cudaStream_t stream);

struct BackwardKernelArgs {
  const uint16_t* rel;       // bf16 bits
  const uint16_t* out;       // forward output O
  const uint16_t* dout;      // incoming gradient dO
  const float* lse;          // forward natural-log LSE, [h * lse_sh + token * lse_st]
  float* delta;              // workspace [n_heads, total_q]: rowsum(dO * O)
  long long total_k;         // rows of k / v / dk / dv (index checks of debug builds)
  uint16_t* dq;
  uint16_t* dk;
  uint16_t* dv;
  uint16_t* drel;
  const int32_t* cu_q;
  const int32_t* cu_k;
  long long rel_st, rel_sh, out_st, out_sh, dout_st, dout_sh, lse_sh, lse_st;
  long long dq_st, dq_sh, dk_st, dk_sh, dv_st, dv_sh, drel_st, drel_sh;
  long long total_q;
  int batch, n_heads, kv_heads, rel_extent;
  int causal, window_left, align_bottom_right;
  float scale;               // softmax_scale
  float scale_log2;          // softmax_scale * log2(e)
  int bias_vec;              // rel 16-byte aligned and rel_extent % 8 == 0 (vector bias windows)
  int slots_first_dkdv;      // dK/dV grid (key slots, kv heads, sequences) instead of
                             // (kv heads, sequences, key slots)
  int slots_first_dq;        // dQ grid (query slots, heads, sequences) instead of
                             // (heads, sequences, query slots)
  int* status;
};

// rel_logits producer: rel[t, h, e] = bf16(tau(pos_t) * sum_j r[t, h, j] * W_h[j, e]).
struct RelLogitsKernelArgs {
  const uint16_t* r;         // bf16 bits, r[t * r_st + h * r_sh + j], j < 16
  const uint16_t* w;         // bf16 bits, W_h[j, e] at w[h * w_sh + j * w_sj + e]
  const int32_t* cu_q;       // optional (null: one sequence)
  const int32_t* cu_k;       // optional (null: positions start at 0)
  long long r_st, r_sh, w_sh, w_sj;
  long long total_q;
  long long units;           // quads: token tiles x head_quads x col_blocks
  int batch, n_heads, rel_extent;
  int head_quads;            // ceil(n_heads / 4)
  int col_blocks;            // ceil(rel_extent / 128)
  float alpha, nf;
  int* status;
};

// Grid of `grid` CTAs (up to kRelLogitsCtasPerSm per SM) striding over args.units quads of
// 128 tokens x 4 heads x 128 columns; rel written through tm_rel ({rel_extent, n_heads, total_q},
// 64 x 1 x 128 boxes, 128-byte swizzle).
cudaError_t launch_rel_logits_sm100(const RelLogitsKernelArgs& args, const CUtensorMap& tm_rel,
                                    int grid, cudaStream_t stream);
constexpr int kRelLogitsCtasPerSm = 4;

// Prep (Delta, zeroed d rel band), dK/dV (+ d rel) and dQ kernels, in that order on `stream`.
cudaError_t launch_backward_sm100(const BackwardKernelArgs& args, const CUtensorMap& tm_q,
                                  const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                                  const CUtensorMap& tm_do, int q_slots, int k_slots,
                                  cudaStream_t stream);

}  // namespace ifa4
