// torch operators over the C ABI: inkling_fa4::prefill_ and decode_; and (at the end of the file) the
// Python calls of the operators next to the attention.
//
// The Python package checks its arguments (the reference's call surface and error messages) and
// then calls one of these operators, which fills the IFA4 parameter block from the tensors'
// pointers and element strides, takes torch's current CUDA stream of the tensors' device, sizes
// and allocates the workspace through torch's caching allocator when the launch needs one, and
// calls ifa4_prefill_launch_ws / ifa4_decode_launch.  This replaces about forty ctypes field
// assignments and two foreign calls per attention call with one dispatcher call (the host cost
// that bounds small launches).  The operators return the C ABI's status code; the caller turns a
// nonzero code into an exception with ifa4_last_error_string().
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/record_function.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

#include <vector>

#include "../../include/inkling_fa4.h"

namespace {

void fill_common(IFA4PrefillParams* p, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                 const at::Tensor& rel, const at::Tensor& out, const at::Tensor& cu_q,
                 const at::Tensor& cu_k, const c10::optional<at::Tensor>& block_table,
                 int64_t rel_extent, bool causal, int64_t window_left, int64_t causal_align) {
  p->q = q.data_ptr();
  p->k = k.data_ptr();
  p->v = v.data_ptr();
  p->rel = rel.data_ptr();
  p->out = out.data_ptr();
  p->cu_seqlens_q = static_cast<const int32_t*>(cu_q.data_ptr());
  p->cu_seqlens_k = static_cast<const int32_t*>(cu_k.data_ptr());
  p->q_stride_t = q.stride(0);
  p->q_stride_h = q.stride(1);
  p->k_stride_t = k.stride(-3);
  p->k_stride_h = k.stride(-2);
  p->v_stride_t = v.stride(-3);
  p->v_stride_h = v.stride(-2);
  p->rel_stride_t = rel.stride(0);
  p->rel_stride_h = rel.stride(1);
  p->out_stride_t = out.stride(0);
  p->out_stride_h = out.stride(1);
  p->total_q = q.size(0);
  p->batch = static_cast<int32_t>(cu_q.numel() - 1);
  p->n_heads = static_cast<int32_t>(q.size(1));
  p->kv_heads = static_cast<int32_t>(k.size(-2));
  p->head_dim = 128;
  p->rel_extent = static_cast<int32_t>(rel_extent);
  p->causal = causal ? 1 : 0;
  p->window_left = static_cast<int32_t>(window_left);
  p->causal_align = static_cast<int32_t>(causal_align);
  p->dtype = IFA4_DTYPE_BF16;
  if (block_table.has_value()) {
    const at::Tensor& bt = *block_table;
    p->total_k = k.size(0) * k.size(1);
    p->block_table = static_cast<const int32_t*>(bt.data_ptr());
    p->block_table_stride = bt.stride(0);
    p->k_stride_page = k.stride(0);
    p->v_stride_page = v.stride(0);
    p->page_size = static_cast<int32_t>(k.size(1));
    p->num_pages = static_cast<int32_t>(k.size(0));
  } else {
    p->total_k = k.size(0);
  }
}

int64_t prefill_op(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                   const at::Tensor& rel, const at::Tensor& out, const at::Tensor& cu_q,
                   const at::Tensor& cu_k, const c10::optional<at::Tensor>& lse,
                   const c10::optional<at::Tensor>& block_table,
                   const c10::optional<at::Tensor>& workspace, int64_t rel_extent, bool causal,
                   int64_t window_left, int64_t causal_align, int64_t max_seqlen_q,
                   int64_t max_seqlen_k, double softmax_scale, int64_t tile_config,
                   int64_t kv_splits) {
  const c10::cuda::CUDAGuard guard(q.device());
  IFA4PrefillParams p{};
  fill_common(&p, q, k, v, rel, out, cu_q, cu_k, block_table, rel_extent, causal, window_left,
              causal_align);
  if (lse.has_value()) {
    p.lse = static_cast<float*>(lse->data_ptr());
    p.lse_stride_h = lse->stride(0);
    p.lse_stride_t = lse->stride(1);
  }
  p.max_seqlen_q = static_cast<int32_t>(max_seqlen_q);
  p.max_seqlen_k = static_cast<int32_t>(max_seqlen_k);
  p.softmax_scale = static_cast<float>(softmax_scale);
  p.tile_config = static_cast<int32_t>(tile_config);
  p.kv_splits = static_cast<int32_t>(kv_splits);
  void* stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  if (p.kv_splits == 1) return ifa4_prefill_launch(&p, stream);
  size_t need = 0;
  int rc = ifa4_prefill_workspace_size(&p, &need);
  if (rc) return rc;
  at::Tensor ws;
  if (need > 0) {
    if (workspace.has_value() && static_cast<size_t>(workspace->nbytes()) >= need)
      ws = *workspace;
    else
      ws = at::empty({static_cast<int64_t>(need)}, q.options().dtype(at::kByte));
  }
  return ifa4_prefill_launch_ws(&p, need > 0 ? ws.data_ptr() : nullptr, need, stream);
}

IFA4DecodeParams decode_params(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               const at::Tensor& rel, const at::Tensor& out,
                               const at::Tensor& cu_q, const at::Tensor& cu_k,
                               const c10::optional<at::Tensor>& lse,
                               const c10::optional<at::Tensor>& block_table, int64_t rel_extent,
                               bool causal, int64_t window_left, int64_t causal_align,
                               int64_t max_seqlen_k, double softmax_scale, int64_t num_splits,
                               int64_t chunk_len) {
  // the decode parameter block starts with the same fields as the prefill one
  IFA4PrefillParams common{};
  fill_common(&common, q, k, v, rel, out, cu_q, cu_k, block_table, rel_extent, causal,
              window_left, causal_align);
  IFA4DecodeParams p{};
  p.q = common.q;
  p.k = common.k;
  p.v = common.v;
  p.rel = common.rel;
  p.out = common.out;
  p.cu_seqlens_q = common.cu_seqlens_q;
  p.cu_seqlens_k = common.cu_seqlens_k;
  p.q_stride_t = common.q_stride_t;
  p.q_stride_h = common.q_stride_h;
  p.k_stride_t = common.k_stride_t;
  p.k_stride_h = common.k_stride_h;
  p.v_stride_t = common.v_stride_t;
  p.v_stride_h = common.v_stride_h;
  p.rel_stride_t = common.rel_stride_t;
  p.rel_stride_h = common.rel_stride_h;
  p.out_stride_t = common.out_stride_t;
  p.out_stride_h = common.out_stride_h;
  p.total_q = common.total_q;
  p.total_k = common.total_k;
  p.batch = common.batch;
  p.n_heads = common.n_heads;
  p.kv_heads = common.kv_heads;
  p.head_dim = common.head_dim;
  p.rel_extent = common.rel_extent;
  p.causal = common.causal;
  p.window_left = common.window_left;
  p.causal_align = common.causal_align;
  p.dtype = common.dtype;
  p.block_table = common.block_table;
  p.block_table_stride = common.block_table_stride;
  p.k_stride_page = common.k_stride_page;
  p.v_stride_page = common.v_stride_page;
  p.page_size = common.page_size;
  p.num_pages = common.num_pages;
  if (lse.has_value()) {
    p.lse = static_cast<float*>(lse->data_ptr());
    p.lse_stride_h = lse->stride(0);
    p.lse_stride_t = lse->stride(1);
  }
  p.max_seqlen_k = static_cast<int32_t>(max_seqlen_k);
  p.softmax_scale = static_cast<float>(softmax_scale);
  p.num_splits = static_cast<int32_t>(num_splits);
  p.chunk_len = static_cast<int32_t>(chunk_len);
  return p;
}

int64_t decode_op(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor& rel, const at::Tensor& out, const at::Tensor& cu_q,
                  const at::Tensor& cu_k, const c10::optional<at::Tensor>& lse,
                  const c10::optional<at::Tensor>& block_table,
                  const c10::optional<at::Tensor>& workspace, int64_t rel_extent, bool causal,
                  int64_t window_left, int64_t causal_align, int64_t max_seqlen_k,
                  double softmax_scale, int64_t num_splits, int64_t chunk_len) {
  const c10::cuda::CUDAGuard guard(q.device());
  const IFA4DecodeParams p = decode_params(q, k, v, rel, out, cu_q, cu_k, lse, block_table,
                                           rel_extent, causal, window_left, causal_align,
                                           max_seqlen_k, softmax_scale, num_splits, chunk_len);
  void* stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  size_t need = 0;
  int rc = ifa4_decode_workspace_size(&p, &need, nullptr, nullptr);
  if (rc) return rc;
  at::Tensor ws;
  if (need > 0) {
    if (workspace.has_value() && static_cast<size_t>(workspace->nbytes()) >= need)
      ws = *workspace;
    else
      ws = at::empty({static_cast<int64_t>(need)}, q.options().dtype(at::kByte));
  }
  return ifa4_decode_launch(&p, need > 0 ? ws.data_ptr() : nullptr,
                            need > 0 ? static_cast<size_t>(ws.nbytes()) : 0, stream);
}

// ---------------------------------------------------------------------------------------------
// Operators next to the attention.  Each takes the arguments of its Python entry point as they are,
// decides whether they are the plain case (types, shapes, one device, layouts the kernels read in
// place), allocates the outputs, launches and returns them; anything else, failed launches among it,
// returns nothing, and the entry point then goes through its own checks and the C ABI, which copy
// what has to be copied and say what is wrong.  They are plain Python functions (the table at the end
// of the file), not dispatcher operators: they have one implementation and no autograd formula, and
// a small call costs the host more than the device.  Norm and rotation of 128 tokens: 5.4 us of host
// time a call, 8.2 as a dispatcher operator (whose argument matching and boxing took 2 us); the append
// of one token 6.0 us with its Python part, 11 before.
// ---------------------------------------------------------------------------------------------
typedef std::vector<at::Tensor> Tensors;
typedef c10::optional<at::Tensor> MaybeTensor;

const void* ptr_or_null(const MaybeTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }
bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
void* stream_of(const at::Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}
at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt));
}
at::Tensor bytes_like(const at::Tensor& t, size_t n) {
  return new_tensor({static_cast<int64_t>(n)}, at::kByte, t);
}
at::Tensor rows_like(const at::Tensor& t) {  // contiguous, same sizes
  return new_tensor(t.sizes(), at::kBFloat16, t);
}

// A caller's tensor was written: autograd refuses a backward that saved its old values.  (Tensors of
// inference mode have no version.)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// [tokens, heads, 128] bf16 rows the kernels read in place.
bool plain_rows(const at::Tensor& t, const at::Tensor& like) {
  return t.is_cuda() && t.dim() == 3 && t.size(2) == 128 && t.scalar_type() == at::kBFloat16 &&
         t.device() == like.device() && t.size(0) == like.size(0) && t.stride(2) == 1 &&
         t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && aligned16(t);
}
bool plain_cu(const MaybeTensor& t, const at::Tensor& like) {
  return !t.has_value() || (t->dim() == 1 && t->numel() >= 2 && t->scalar_type() == at::kInt &&
                            t->device() == like.device() && t->stride(0) == 1);
}
bool plain_weight(const MaybeTensor& t, const at::Tensor& like) {
  return !t.has_value() ||
         (t->dim() == 1 && t->numel() == 128 && t->stride(0) == 1 && t->device() == like.device() &&
          (t->scalar_type() == at::kBFloat16 || t->scalar_type() == at::kFloat));
}
// The step's other arguments.  eps -1: no norm; any other value that is not >= 0 (NaN stands for
// what the Python checks have to look at) is not the plain case.
bool plain_step(const at::Tensor& like, const MaybeTensor& q_weight, const MaybeTensor& k_weight,
                const MaybeTensor& inv_freq, const MaybeTensor& cu_q, const MaybeTensor& cu_k,
                double eps) {
  if (!(eps >= 0) && eps != -1.0) return false;
  if (!plain_cu(cu_q, like) || !plain_cu(cu_k, like) || !plain_weight(q_weight, like) ||
      !plain_weight(k_weight, like))
    return false;
  if (cu_k.has_value() && (!cu_q.has_value() || cu_k->numel() != cu_q->numel())) return false;
  if (q_weight.has_value() && k_weight.has_value() &&
      q_weight->scalar_type() != k_weight->scalar_type())
    return false;
  if (!(eps >= 0) && (q_weight.has_value() || k_weight.has_value())) return false;
  if (!inv_freq.has_value()) return true;
  return inv_freq->dim() == 1 && inv_freq->numel() > 0 && inv_freq->numel() <= 64 &&
         inv_freq->numel() % 8 == 0 && inv_freq->stride(0) == 1 &&
         inv_freq->device() == like.device() &&
         (inv_freq->scalar_type() == at::kDouble || inv_freq->scalar_type() == at::kFloat);
}

// The fields the norm-and-rotation parameter blocks share.
template <class P>
void fill_norm_rope(P* p, const MaybeTensor& q_weight, const MaybeTensor& k_weight,
                    const MaybeTensor& inv_freq, const MaybeTensor& cu_q, const MaybeTensor& cu_k,
                    int64_t total_q, int64_t heads, int64_t kv_heads, bool interleaved,
                    double eps) {
  p->q_weight = ptr_or_null(q_weight);
  p->k_weight = ptr_or_null(k_weight);
  p->inv_freq = ptr_or_null(inv_freq);
  p->cu_seqlens_q = static_cast<const int32_t*>(ptr_or_null(cu_q));
  p->cu_seqlens_k = static_cast<const int32_t*>(ptr_or_null(cu_k));
  p->total_q = total_q;
  p->batch = cu_q.has_value() ? static_cast<int32_t>(cu_q->numel() - 1) : 1;
  p->n_heads = static_cast<int32_t>(heads);
  p->kv_heads = static_cast<int32_t>(kv_heads);
  p->head_dim = 128;
  p->rotary_dim = inv_freq.has_value() ? static_cast<int32_t>(2 * inv_freq->numel()) : 0;
  p->interleaved = interleaved;
  p->normalize = eps >= 0;
  const MaybeTensor& w = q_weight.has_value() ? q_weight : k_weight;
  p->weight_dtype = w.has_value() && w->scalar_type() == at::kFloat ? IFA4_WEIGHT_F32
                                                                    : IFA4_WEIGHT_BF16;
  p->inv_freq_f32 = inv_freq.has_value() && inv_freq->scalar_type() == at::kFloat;
  p->dtype = IFA4_DTYPE_BF16;
  p->eps = eps >= 0 ? static_cast<float>(eps) : 0.f;
}

Tensors qk_norm_rope_op(const at::Tensor& q, const at::Tensor& k, const MaybeTensor& q_weight,
                        const MaybeTensor& k_weight, const MaybeTensor& inv_freq,
                        const MaybeTensor& cu_q, const MaybeTensor& cu_k, bool interleaved,
                        double eps) {
  if (!plain_rows(q, q) || !plain_rows(k, q) || !(eps >= 0 || inv_freq.has_value()) ||
      !plain_step(q, q_weight, k_weight, inv_freq, cu_q, cu_k, eps))
    return {};
  const c10::cuda::CUDAGuard guard(q.device());
  const at::Tensor q_out = rows_like(q), k_out = rows_like(k);
  IFA4QkNormRopeParams p{};
  fill_norm_rope(&p, q_weight, k_weight, inv_freq, cu_q, cu_k, q.size(0), q.size(1), k.size(1),
                 interleaved, eps);
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.q_out = q_out.data_ptr();
  p.k_out = k_out.data_ptr();
  p.q_stride_t = q.stride(0);
  p.q_stride_h = q.stride(1);
  p.k_stride_t = k.stride(0);
  p.k_stride_h = k.stride(1);
  p.q_out_stride_t = q_out.stride(0);
  p.q_out_stride_h = q_out.stride(1);
  p.k_out_stride_t = k_out.stride(0);
  p.k_out_stride_h = k_out.stride(1);
  p.zero_padding = 1;
  if (ifa4_qk_norm_rope_launch(&p, stream_of(q))) return {};
  return {q_out, k_out};
}

// Returns dq, dk and the gradients of the weights that are there and wanted.
Tensors qk_norm_rope_backward_op(const at::Tensor& dq_out, const at::Tensor& dk_out,
                                 const at::Tensor& q, const at::Tensor& k,
                                 const MaybeTensor& q_weight, const MaybeTensor& k_weight,
                                 const MaybeTensor& inv_freq, const MaybeTensor& cu_q,
                                 const MaybeTensor& cu_k, bool interleaved, double eps,
                                 bool want_q_weight, bool want_k_weight) {
  if (!plain_rows(q, q) || !plain_rows(k, q) || !plain_rows(dq_out, q) || !plain_rows(dk_out, q) ||
      dq_out.size(1) != q.size(1) || dk_out.size(1) != k.size(1) ||
      !plain_step(q, q_weight, k_weight, inv_freq, cu_q, cu_k, eps))
    return {};
  const c10::cuda::CUDAGuard guard(q.device());
  Tensors out{rows_like(q), rows_like(k)};
  IFA4QkNormRopeBackwardParams p{};
  fill_norm_rope(&p, q_weight, k_weight, inv_freq, cu_q, cu_k, q.size(0), q.size(1), k.size(1),
                 interleaved, eps);
  if (q_weight.has_value() && want_q_weight) {
    out.push_back(new_tensor({128}, q_weight->scalar_type(), q));
    p.dq_weight = out.back().data_ptr();
  }
  if (k_weight.has_value() && want_k_weight) {
    out.push_back(new_tensor({128}, k_weight->scalar_type(), q));
    p.dk_weight = out.back().data_ptr();
  }
  p.dq_out = dq_out.data_ptr();
  p.dk_out = dk_out.data_ptr();
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.dq = out[0].data_ptr();
  p.dk = out[1].data_ptr();
  p.dq_out_stride_t = dq_out.stride(0);
  p.dq_out_stride_h = dq_out.stride(1);
  p.dk_out_stride_t = dk_out.stride(0);
  p.dk_out_stride_h = dk_out.stride(1);
  p.q_stride_t = q.stride(0);
  p.q_stride_h = q.stride(1);
  p.k_stride_t = k.stride(0);
  p.k_stride_h = k.stride(1);
  p.dq_stride_t = out[0].stride(0);
  p.dq_stride_h = out[0].stride(1);
  p.dk_stride_t = out[1].stride(0);
  p.dk_stride_h = out[1].stride(1);
  size_t need = 0;
  if (ifa4_qk_norm_rope_backward_workspace_size(&p, &need)) return {};
  at::Tensor ws;
  if (need > 0) ws = bytes_like(q, need);
  if (ifa4_qk_norm_rope_backward_launch(&p, need > 0 ? ws.data_ptr() : nullptr, need, stream_of(q)))
    return {};
  return out;
}

// The append with its queries; returns q_out.
Tensors kv_append_op(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                     const at::Tensor& k_cache, const at::Tensor& v_cache,
                     const MaybeTensor& q_weight, const MaybeTensor& k_weight,
                     const MaybeTensor& inv_freq, const at::Tensor& cu_q, const at::Tensor& cu_k,
                     const at::Tensor& block_table, bool interleaved, double eps) {
  if (!plain_rows(k, k) || !plain_rows(v, k) || !plain_rows(q, k) || v.size(1) != k.size(1) ||
      !plain_step(k, q_weight, k_weight, inv_freq, cu_q, cu_k, eps))
    return {};
  for (const at::Tensor* c : {&k_cache, &v_cache})
    if (c->dim() != 4 || c->scalar_type() != at::kBFloat16 || c->device() != k.device() ||
        c->size(2) != k.size(1) || c->size(3) != 128 || c->stride(3) != 1 || !aligned16(*c))
      return {};
  for (int i = 0; i < 3; ++i)
    if (k_cache.stride(i) <= 0 || k_cache.stride(i) % 8 != 0 || v_cache.stride(i) <= 0 ||
        v_cache.stride(i) % 8 != 0)
      return {};
  const int64_t page_size = k_cache.size(1);
  if (v_cache.sizes() != k_cache.sizes() || k_cache.data_ptr() == v_cache.data_ptr() ||
      page_size < 16 || (page_size & (page_size - 1)) != 0 || block_table.dim() != 2 ||
      block_table.scalar_type() != at::kInt || block_table.device() != k.device() ||
      block_table.size(0) != cu_q.numel() - 1 || block_table.numel() == 0 ||
      block_table.stride(1) != 1)
    return {};
  const c10::cuda::CUDAGuard guard(k.device());
  const at::Tensor q_out = rows_like(q);
  IFA4KvAppendParams p{};
  fill_norm_rope(&p, q_weight, k_weight, inv_freq, cu_q, cu_k, k.size(0), q.size(1), k.size(1),
                 interleaved, eps);
  p.q = q.data_ptr();
  p.q_out = q_out.data_ptr();
  p.q_stride_t = q.stride(0);
  p.q_stride_h = q.stride(1);
  p.q_out_stride_t = q_out.stride(0);
  p.q_out_stride_h = q_out.stride(1);
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.k_cache = k_cache.data_ptr();
  p.v_cache = v_cache.data_ptr();
  p.k_stride_t = k.stride(0);
  p.k_stride_h = k.stride(1);
  p.v_stride_t = v.stride(0);
  p.v_stride_h = v.stride(1);
  p.k_stride_page = k_cache.stride(0);
  p.k_cache_stride_t = k_cache.stride(1);
  p.k_cache_stride_h = k_cache.stride(2);
  p.v_stride_page = v_cache.stride(0);
  p.v_cache_stride_t = v_cache.stride(1);
  p.v_cache_stride_h = v_cache.stride(2);
  p.block_table = static_cast<const int32_t*>(block_table.data_ptr());
  p.block_table_stride = block_table.stride(0);
  p.zero_padding = 1;
  p.page_size = static_cast<int32_t>(page_size);
  p.num_pages = static_cast<int32_t>(k_cache.size(0));
  p.table_width = static_cast<int32_t>(block_table.size(1));
  if (ifa4_kv_append_launch(&p, stream_of(k))) return {};
  written(k_cache);
  written(v_cache);
  return {q_out};
}

// Returns out.
Tensors decode_shared_prefix_op(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                const at::Tensor& rel, const at::Tensor& cu_q,
                                const at::Tensor& cu_k, const at::Tensor& block_table,
                                const MaybeTensor& workspace, int64_t rel_extent,
                                int64_t window_left, int64_t max_seqlen_k, double softmax_scale,
                                int64_t num_splits, int64_t chunk_len, int64_t shared_prefix_len,
                                int64_t prefix_splits) {
  auto outer_ok = [](const at::Tensor& t) {
    for (int64_t i = 0; i + 1 < t.dim(); ++i)
      if (t.stride(i) <= 0 || t.stride(i) % 8 != 0) return false;
    return t.stride(t.dim() - 1) == 1 && aligned16(t);
  };
  if (!plain_rows(q, q) || !outer_ok(q) || k.dim() != 4 || v.sizes() != k.sizes() ||
      k.size(3) != 128 || k.scalar_type() != at::kBFloat16 || v.scalar_type() != at::kBFloat16 ||
      k.device() != q.device() || v.device() != q.device() || !outer_ok(k) || !outer_ok(v) ||
      !plain_cu(cu_q, q) || !plain_cu(cu_k, q) || cu_k.numel() != cu_q.numel() ||
      q.size(0) != cu_q.numel() - 1 || rel.dim() != 3 || rel.scalar_type() != at::kBFloat16 ||
      rel.device() != q.device() || rel.size(0) != q.size(0) || rel.size(1) != q.size(1) ||
      rel.stride(2) != 1 || rel_extent < 1 || rel_extent > rel.size(2) || k.size(2) < 1 ||
      q.size(1) % k.size(2) != 0)
    return {};
  const int64_t page_size = k.size(1);
  if (page_size < 16 || (page_size & (page_size - 1)) != 0 || block_table.dim() != 2 ||
      block_table.scalar_type() != at::kInt || block_table.device() != q.device() ||
      block_table.size(0) != q.size(0) || block_table.numel() == 0 || block_table.stride(1) != 1 ||
      shared_prefix_len < 0 || shared_prefix_len > block_table.size(1) * page_size ||
      shared_prefix_len > (1 << 30) || !(softmax_scale > 0))
    return {};
  for (int64_t x : {window_left, max_seqlen_k, num_splits, chunk_len, prefix_splits})
    if (x < -1 || x > 0x7fffffff) return {};
  const c10::cuda::CUDAGuard guard(q.device());
  const at::Tensor out = rows_like(q);
  IFA4SharedPrefixParams p{};
  p.decode = decode_params(q, k, v, rel, out, cu_q, cu_k, c10::nullopt, block_table, rel_extent,
                           true, window_left, IFA4_ALIGN_BOTTOM_RIGHT, max_seqlen_k, softmax_scale,
                           num_splits, chunk_len);
  p.shared_prefix_len = static_cast<int32_t>(shared_prefix_len);
  p.prefix_splits = static_cast<int32_t>(prefix_splits);
  size_t need = 0;
  if (ifa4_decode_shared_prefix_workspace_size(&p, &need)) return {};
  at::Tensor ws;
  if (workspace.has_value() && (workspace->device() != q.device() || !workspace->is_contiguous()))
    return {};
  if (need > 0)
    ws = workspace.has_value() && static_cast<size_t>(workspace->nbytes()) >= need
             ? *workspace : bytes_like(q, need);
  if (ifa4_decode_shared_prefix_launch(&p, need > 0 ? ws.data_ptr() : nullptr, need, stream_of(q)))
    return {};
  return {out};
}

int32_t weight_dtype(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat ? IFA4_WEIGHT_F32 : IFA4_WEIGHT_BF16;
}
bool plain_starts(const at::Tensor& starts, const at::Tensor& like) {
  return starts.dim() == 1 && starts.scalar_type() == at::kInt && starts.numel() >= 1 &&
         starts.numel() <= IFA4_MAX_BUCKETS && starts.device() == like.device() &&
         starts.stride(0) == 1;
}

Tensors bucket_bias_op(const at::Tensor& table, const at::Tensor& starts, int64_t total_q,
                       int64_t rel_extent) {
  if (!table.is_cuda() || table.dim() != 2 || (table.scalar_type() != at::kFloat && table.scalar_type() != at::kBFloat16) ||
      !plain_starts(starts, table) || table.size(0) != starts.numel() || table.size(1) < 1 ||
      total_q < 0 || rel_extent < 1 || rel_extent > (1 << 24))
    return {};
  const c10::cuda::CUDAGuard guard(table.device());
  const int64_t heads = table.size(1);
  const at::Tensor rel = new_tensor({heads, rel_extent}, at::kBFloat16, table);
  IFA4BucketBiasParams p{};
  p.table = table.data_ptr();
  p.starts = static_cast<const int32_t*>(starts.data_ptr());
  p.rel = rel.data_ptr();
  p.table_stride_b = table.stride(0);
  p.table_stride_h = table.stride(1);
  p.rel_stride_h = rel.stride(0);
  p.n_heads = static_cast<int32_t>(heads);
  p.rel_extent = static_cast<int32_t>(rel_extent);
  p.buckets = static_cast<int32_t>(starts.numel());
  p.weight_dtype = weight_dtype(table);
  if (ifa4_bucket_bias_launch(&p, stream_of(table))) return {};
  // the tokens of rel_logits are the same memory
  const int64_t sizes[] = {total_q, heads, rel_extent}, strides[] = {0, rel_extent, 1};
  rel.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef(sizes), at::IntArrayRef(strides));
  return {rel};
}

Tensors bucket_bias_backward_op(const at::Tensor& drel, const at::Tensor& starts, bool f32,
                                const MaybeTensor& cu_q) {
  if (!drel.is_cuda() || drel.dim() != 3 || drel.scalar_type() != at::kBFloat16 || drel.size(1) < 1 ||
      drel.size(2) < 1 || drel.size(2) > (1 << 24) || (drel.size(2) > 1 && drel.stride(2) != 1) ||
      !plain_starts(starts, drel))
    return {};
  if (cu_q.has_value() && (cu_q->dim() != 1 || cu_q->numel() < 1 || cu_q->scalar_type() != at::kInt ||
                           cu_q->device() != drel.device() || cu_q->stride(0) != 1))
    return {};
  const c10::cuda::CUDAGuard guard(drel.device());
  const at::Tensor dtable = new_tensor({starts.numel(), drel.size(1)},
                                       f32 ? at::kFloat : at::kBFloat16, drel);
  IFA4BucketBiasBackwardParams p{};
  p.drel = drel.data_ptr();
  p.starts = static_cast<const int32_t*>(starts.data_ptr());
  p.cu_seqlens_q = static_cast<const int32_t*>(ptr_or_null(cu_q));
  p.dtable = dtable.data_ptr();
  p.drel_stride_t = drel.stride(0);
  p.drel_stride_h = drel.stride(1);
  p.dtable_stride_b = dtable.stride(0);
  p.dtable_stride_h = dtable.stride(1);
  p.total_q = drel.size(0);
  p.batch = cu_q.has_value() ? static_cast<int32_t>(cu_q->numel() - 1) : 0;
  p.n_heads = static_cast<int32_t>(drel.size(1));
  p.rel_extent = static_cast<int32_t>(drel.size(2));
  p.buckets = static_cast<int32_t>(starts.numel());
  p.weight_dtype = f32 ? IFA4_WEIGHT_F32 : IFA4_WEIGHT_BF16;
  size_t need = 0;
  if (ifa4_bucket_bias_backward_workspace_size(&p, &need)) return {};
  at::Tensor ws;
  if (need > 0) ws = bytes_like(drel, need);
  if (ifa4_bucket_bias_backward_launch(&p, need > 0 ? ws.data_ptr() : nullptr, need,
                                       stream_of(drel)))
    return {};
  return {dtable};
}

// ---------------------------------------------------------------------------------------------
// The same as Python functions: positional arguments; a tuple of tensors, or None.
// ---------------------------------------------------------------------------------------------
struct Arguments {
  PyObject* const* objects;
  Py_ssize_t count;
  Py_ssize_t next = 0;
  bool ok = true;  // false: a type that is not the plain case

  PyObject* take() {
    if (next < count) return objects[next++];
    ok = false;
    return Py_None;
  }
  at::Tensor tensor_of(PyObject* o) {
    if (THPVariable_Check(o)) return THPVariable_Unpack(o);
    ok = false;
    return at::Tensor();
  }
  at::Tensor tensor() { return tensor_of(take()); }
  MaybeTensor maybe() {
    PyObject* o = take();
    if (o == Py_None) return c10::nullopt;
    return tensor_of(o);
  }
  bool flag() {
    PyObject* o = take();
    ok = ok && PyBool_Check(o);
    return o == Py_True;
  }
  int64_t integer() {
    PyObject* o = take();
    int overflow = 0;
    if (!PyLong_Check(o)) {
      ok = false;
      return 0;
    }
    const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
    ok = ok && overflow == 0;
    return v;
  }
  double real() {
    PyObject* o = take();
    ok = ok && PyFloat_Check(o);
    return ok ? PyFloat_AS_DOUBLE(o) : 0.0;
  }
  bool complete() const { return ok && next == count; }
};

// Other Python threads run while this one allocates and launches.
struct WithoutGil {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

// Reads the arguments (`read`, which returns the work) and does the work.
template <class Read>
PyObject* call(const char* name, PyObject* const* objects, Py_ssize_t count, Read read) {
  Tensors out;
  // A dispatch mode or a tracer does not see what these functions do; the checks refuse a tracer.
  if (c10::impl::TorchDispatchModeTLS::any_modes_set() || at::tracer::impl::is_dispatch_enabled())
    Py_RETURN_NONE;
  try {
    RECORD_FUNCTION(name, c10::ArrayRef<const c10::IValue>{});
    Arguments a{objects, count};
    auto work = read(a);
    if (a.complete()) {
      WithoutGil no_gil;
      out = work();
    }
  } catch (const std::exception&) {  // an allocation, a tensor without memory: the checks say it
    out.clear();
  }
  if (out.empty()) Py_RETURN_NONE;
  PyObject* result = PyTuple_New(static_cast<Py_ssize_t>(out.size()));
  if (result == nullptr) return nullptr;
  for (size_t i = 0; i < out.size(); ++i) {
    PyObject* o = THPVariable_Wrap(std::move(out[i]));
    if (o == nullptr) {
      Py_DECREF(result);
      return nullptr;
    }
    PyTuple_SET_ITEM(result, static_cast<Py_ssize_t>(i), o);
  }
  return result;
}

PyObject* py_qk_norm_rope(PyObject*, PyObject* const* objects, Py_ssize_t count) {
  return call("inkling_fa4::qk_norm_rope", objects, count, [](Arguments& a) {
    auto q = a.tensor(), k = a.tensor();
    auto wq = a.maybe(), wk = a.maybe(), inv_freq = a.maybe(), cu_q = a.maybe(), cu_k = a.maybe();
    const bool interleaved = a.flag();
    const double eps = a.real();
    return [=] { return qk_norm_rope_op(q, k, wq, wk, inv_freq, cu_q, cu_k, interleaved, eps); };
  });
}

PyObject* py_qk_norm_rope_backward(PyObject*, PyObject* const* objects, Py_ssize_t count) {
  return call("inkling_fa4::qk_norm_rope_backward", objects, count, [](Arguments& a) {
    auto dq_out = a.tensor(), dk_out = a.tensor(), q = a.tensor(), k = a.tensor();
    auto wq = a.maybe(), wk = a.maybe(), inv_freq = a.maybe(), cu_q = a.maybe(), cu_k = a.maybe();
    const bool interleaved = a.flag();
    const double eps = a.real();
    const bool want_q = a.flag(), want_k = a.flag();
    return [=] {
      return qk_norm_rope_backward_op(dq_out, dk_out, q, k, wq, wk, inv_freq, cu_q, cu_k,
                                      interleaved, eps, want_q, want_k);
    };
  });
}

PyObject* py_kv_append(PyObject*, PyObject* const* objects, Py_ssize_t count) {
  return call("inkling_fa4::kv_append", objects, count, [](Arguments& a) {
    auto q = a.tensor(), k = a.tensor(), v = a.tensor();
    auto k_cache = a.tensor(), v_cache = a.tensor();
    auto wq = a.maybe(), wk = a.maybe(), inv_freq = a.maybe();
    auto cu_q = a.tensor(), cu_k = a.tensor(), block_table = a.tensor();
    const bool interleaved = a.flag();
    const double eps = a.real();
    return [=] {
      return kv_append_op(q, k, v, k_cache, v_cache, wq, wk, inv_freq, cu_q, cu_k, block_table,
                          interleaved, eps);
    };
  });
}

PyObject* py_decode_shared_prefix(PyObject*, PyObject* const* objects, Py_ssize_t count) {
  return call("inkling_fa4::decode_shared_prefix", objects, count, [](Arguments& a) {
    auto q = a.tensor(), k = a.tensor(), v = a.tensor(), rel = a.tensor();
    auto cu_q = a.tensor(), cu_k = a.tensor(), block_table = a.tensor();
    auto workspace = a.maybe();
    const int64_t rel_extent = a.integer(), window_left = a.integer(), max_seqlen_k = a.integer();
    const double softmax_scale = a.real();
    const int64_t num_splits = a.integer(), chunk_len = a.integer();
    const int64_t shared_prefix_len = a.integer(), prefix_splits = a.integer();
    return [=] {
      return decode_shared_prefix_op(q, k, v, rel, cu_q, cu_k, block_table, workspace, rel_extent,
                                     window_left, max_seqlen_k, softmax_scale, num_splits,
                                     chunk_len, shared_prefix_len, prefix_splits);
    };
  });
}

PyObject* py_bucket_bias(PyObject*, PyObject* const* objects, Py_ssize_t count) {
  return call("inkling_fa4::bucket_bias", objects, count, [](Arguments& a) {
    auto table = a.tensor(), starts = a.tensor();
    const int64_t total_q = a.integer(), rel_extent = a.integer();
    return [=] { return bucket_bias_op(table, starts, total_q, rel_extent); };
  });
}

PyObject* py_bucket_bias_backward(PyObject*, PyObject* const* objects, Py_ssize_t count) {
  return call("inkling_fa4::bucket_bias_backward", objects, count, [](Arguments& a) {
    auto drel = a.tensor(), starts = a.tensor();
    const bool f32 = a.flag();
    auto cu_q = a.maybe();
    return [=] { return bucket_bias_backward_op(drel, starts, f32, cu_q); };
  });
}

template <class F>
PyMethodDef method(const char* name, F* f) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL,
          nullptr};
}
PyMethodDef kMethods[] = {
    method("qk_norm_rope", py_qk_norm_rope),
    method("qk_norm_rope_backward", py_qk_norm_rope_backward),
    method("kv_append", py_kv_append),
    method("decode_shared_prefix", py_decode_shared_prefix),
    method("bucket_bias", py_bucket_bias),
    method("bucket_bias_backward", py_bucket_bias_backward),
};
}  // namespace

// A dict of the functions above by name (called once, with the GIL held).
extern "C" PyObject* ifa4_python_calls(void) {
  PyObject* calls = PyDict_New();
  if (calls == nullptr) return nullptr;
  for (PyMethodDef& m : kMethods) {
    PyObject* f = PyCFunction_New(&m, nullptr);
    const int rc = f == nullptr ? -1 : PyDict_SetItemString(calls, m.ml_name, f);
    Py_XDECREF(f);
    if (rc != 0) {
      Py_DECREF(calls);
      return nullptr;
    }
  }
  return calls;
}

TORCH_LIBRARY(inkling_fa4, m) {
  m.def("prefill_(Tensor q, Tensor k, Tensor v, Tensor rel, Tensor(a!) out, Tensor cu_q, "
        "Tensor cu_k, Tensor(b!)? lse, Tensor? block_table, Tensor? workspace, int rel_extent, "
        "bool causal, int window_left, int causal_align, int max_seqlen_q, int max_seqlen_k, "
        "float softmax_scale, int tile_config, int kv_splits) -> int");
  m.def("decode_(Tensor q, Tensor k, Tensor v, Tensor rel, Tensor(a!) out, Tensor cu_q, "
        "Tensor cu_k, Tensor(b!)? lse, Tensor? block_table, Tensor? workspace, int rel_extent, "
        "bool causal, int window_left, int causal_align, int max_seqlen_k, float softmax_scale, "
        "int num_splits, int chunk_len) -> int");
}

TORCH_LIBRARY_IMPL(inkling_fa4, CUDA, m) {
  m.impl("prefill_", &prefill_op);
  m.impl("decode_", &decode_op);
}
