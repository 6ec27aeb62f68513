// Host side of the calls a decode step repeats, on torch's C++ tensors: the checks, the output and
// workspace allocations and the argument blocks of anna_mi.h, which took 15 to 60 us a call in Python
// (linear 17 us around a 3.7 us kernel, a packed-cache decode 35 us, the sparse block 65 us).
//
// Every function here takes only the plain case of its Python caller -- tensors of the right types,
// shapes, layouts and device -- and answers None to anything else, without side effects; the caller
// then goes its general way, which converts or refuses as it always did.  Nothing is kept between
// calls: each one reads the tensors it is given.
//
// The library is not linked: Python hands over the addresses of its entry points (bind), so that its
// stamp check and its error text stay in one place.  The stream is an argument (the caller's current
// stream), so no device header is needed.
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>

#include <cstdint>
#include <cstdlib>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "../../include/anna_mi.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

struct Library {
  decltype(&anna_mi_last_error) last_error = nullptr;
  decltype(&anna_mi_int4_linear) int4_linear = nullptr;
  decltype(&anna_mi_decode_num_blocks) decode_num_blocks = nullptr;
  decltype(&anna_mi_gqa_decode_splitkv) gqa_decode_splitkv = nullptr;
  decltype(&anna_mi_tq_decode) tq_decode = nullptr;
  decltype(&anna_mi_tq_store) tq_store = nullptr;
  decltype(&anna_mi_moe_route_small) moe_route_small = nullptr;
  decltype(&anna_mi_moe_gather) moe_gather = nullptr;
  decltype(&anna_mi_moe_router) moe_router = nullptr;
  decltype(&anna_mi_moe_dispatch) moe_dispatch = nullptr;
  decltype(&anna_mi_moe_grouped_int4_mlp) moe_grouped_int4_mlp = nullptr;
  decltype(&anna_mi_moe_combine) moe_combine = nullptr;
  decltype(&anna_mi_moe_prefill_workspace) moe_prefill_workspace = nullptr;
  decltype(&anna_mi_moe_prefill) moe_prefill = nullptr;
  decltype(&anna_mi_paged_fork) paged_fork = nullptr;
  decltype(&anna_mi_paged_free) paged_free = nullptr;
  decltype(&anna_mi_paged_extend) paged_extend = nullptr;
  decltype(&anna_mi_paged_lengths) paged_lengths = nullptr;
  decltype(&anna_mi_paged_span_plan) paged_span_plan = nullptr;
  decltype(&anna_mi_paged_span_fill) paged_span_fill = nullptr;
  decltype(&anna_mi_paged_store) paged_store = nullptr;
  decltype(&anna_mi_paged_read) paged_read = nullptr;
  decltype(&anna_mi_paged_attend) paged_attend = nullptr;
  decltype(&anna_mi_gated_delta_workspace) gated_delta_workspace = nullptr;
  decltype(&anna_mi_gated_delta) gated_delta = nullptr;
  decltype(&anna_mi_causal_conv1d) causal_conv1d = nullptr;
  decltype(&anna_mi_rms_norm) rms_norm = nullptr;
} lib;

void bind(const py::dict& d) {
  auto get = [&](const char* name, auto& fn) {
    fn = reinterpret_cast<std::decay_t<decltype(fn)>>(d[name].cast<uintptr_t>());
  };
  get("anna_mi_last_error", lib.last_error);
  get("anna_mi_int4_linear", lib.int4_linear);
  get("anna_mi_decode_num_blocks", lib.decode_num_blocks);
  get("anna_mi_gqa_decode_splitkv", lib.gqa_decode_splitkv);
  get("anna_mi_tq_decode", lib.tq_decode);
  get("anna_mi_tq_store", lib.tq_store);
  get("anna_mi_moe_route_small", lib.moe_route_small);
  get("anna_mi_moe_gather", lib.moe_gather);
  get("anna_mi_moe_router", lib.moe_router);
  get("anna_mi_moe_dispatch", lib.moe_dispatch);
  get("anna_mi_moe_grouped_int4_mlp", lib.moe_grouped_int4_mlp);
  get("anna_mi_moe_combine", lib.moe_combine);
  get("anna_mi_moe_prefill_workspace", lib.moe_prefill_workspace);
  get("anna_mi_moe_prefill", lib.moe_prefill);
  get("anna_mi_paged_fork", lib.paged_fork);
  get("anna_mi_paged_free", lib.paged_free);
  get("anna_mi_paged_extend", lib.paged_extend);
  get("anna_mi_paged_lengths", lib.paged_lengths);
  get("anna_mi_paged_span_plan", lib.paged_span_plan);
  get("anna_mi_paged_span_fill", lib.paged_span_fill);
  get("anna_mi_paged_store", lib.paged_store);
  get("anna_mi_paged_read", lib.paged_read);
  get("anna_mi_paged_attend", lib.paged_attend);
  get("anna_mi_gated_delta_workspace", lib.gated_delta_workspace);
  get("anna_mi_gated_delta", lib.gated_delta);
  get("anna_mi_causal_conv1d", lib.causal_conv1d);
  get("anna_mi_rms_norm", lib.rms_norm);
}

void check(int rc, const char* name) {
  if (rc != 0)
    throw std::runtime_error(std::string(name) + " failed (" + std::to_string(rc) + "): " + lib.last_error());
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return ANNA_MI_BF16;
    case at::kHalf: return ANNA_MI_F16;
    case at::kFloat: return ANNA_MI_F32;
    default: return -1;
  }
}

// A plain strided tensor with memory of its own on `dev` (not a fake, batched or sparse one)
bool plain(const Tensor& t, const at::Device& dev) {
  return t.defined() && t.layout() == at::kStrided && t.device() == dev && t.has_storage() &&
         t.unsafeGetTensorImpl()->key_set().has(c10::DispatchKey::CUDA) &&
         !t.unsafeGetTensorImpl()->key_set().has(c10::DispatchKey::Python) && !t.is_conj() && !t.is_neg();
}
bool plain(const OptTensor& t, const at::Device& dev) { return !t || plain(*t, dev); }
bool is(const Tensor& t, const at::Device& dev, at::ScalarType dt) {
  return plain(t, dev) && t.scalar_type() == dt && t.is_contiguous();
}

void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
void* stream_ptr(uintptr_t s) { return reinterpret_cast<void*>(s); }

// ---------------------------------------------------------------- int4 linear

// y = x . dequant(W)^T + bias for x [..., K] of the activation dtype (the tensors and conditions of
// fused_ops._check_int4_inputs).  `compute`: the layer's dtype.
OptTensor int4_linear(const Tensor& x, const Tensor& qw, const Tensor& qs, const Tensor& qz, const OptTensor& bias,
                      int64_t group, int64_t out_features, at::ScalarType compute, uintptr_t stream, bool strategies) {
  // a strategy other than the kernels' is the general path's to read
  if (const char* s = strategies ? std::getenv("ANNA_XPU_INT4_MATMUL") : nullptr; s && *s) return std::nullopt;
  const at::Device dev = x.device();
  if (!dev.is_cuda() || !plain(x, dev) || x.dim() < 1 || x.scalar_type() != compute || dtype_code(x) < 0 || x.numel() == 0)
    return std::nullopt;
  if (!is(qw, dev, at::kInt) || !plain(qs, dev) || dtype_code(qs) < 0 || !qs.is_contiguous() || !is(qz, dev, at::kChar))
    return std::nullopt;
  const int64_t K = x.size(-1), rows = x.numel() / K;
  if (qw.dim() != 2 || qs.dim() != 2 || qz.dim() != 2 || group <= 0 || qw.size(0) != out_features ||
      qw.size(1) * 8 < K || qs.size(1) != qw.size(0) || qz.sizes() != qs.sizes() || qs.size(0) * group < K)
    return std::nullopt;
  if (bias && (!plain(bias, dev) || (bias->requires_grad() && at::GradMode::is_enabled()) || bias->scalar_type() != compute || bias->dim() != 1 || bias->size(0) != out_features))
    return std::nullopt;
  int64_t row_stride = K;
  if (x.dim() == 2) {
    if (x.stride(1) != 1 || (rows > 1 && x.stride(0) < K)) return std::nullopt;
    if (rows > 1) row_stride = x.stride(0);
  } else if (!x.is_contiguous()) {
    return std::nullopt;
  }
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  shape.back() = out_features;
  Tensor y = at::empty(shape, x.options().requires_grad(false));
  check(lib.int4_linear(ptr(x), dtype_code(x), rows, K, row_stride, (const int32_t*)ptr(qw), out_features, qw.size(1),
                        ptr(qs), dtype_code(qs), (const int8_t*)ptr(qz), qs.size(0), group, ptr(y), stream_ptr(stream)),
        "anna_mi_int4_linear");
  if (bias) y.add_(bias->detach());
  return y;
}

// ---------------------------------------------------------------- split-KV decode with per-row lengths

anna_mi_view view(const Tensor& t, bool heads_only = false) {
  anna_mi_view v{ptr(t), t.stride(0), t.stride(1), t.stride(2), 0};
  if (!heads_only) v.s3 = t.stride(3);
  return v;
}
// [B, Hq, D] or [B, Hq, 1, D] as [B, Hq, 1, D]
anna_mi_view query_view(const Tensor& t) {
  return t.dim() == 3 ? anna_mi_view{ptr(t), t.stride(0), t.stride(1), 0, t.stride(2)} : view(t);
}

// One decode over [quantized slots ++ window] of every row: keys dense in the query's dtype or TQ-MSE
// codes (key_norms given), values in min/max groups.  query, gate, out: [B, Hq, D] or [B, Hq, 1, D].
// Without partial buffers they are allocated here; None also where given ones hold too few blocks.
OptTensor decode_rows(const Tensor& q, const OptTensor& gate, const OptTensor& out_in, const OptTensor& key,
                      const OptTensor& key_norms, const OptTensor& vdata, const OptTensor& vscales,
                      const OptTensor& vzeros, const Tensor& rk, const Tensor& rv, const Tensor& seq_lengths,
                      const Tensor& rotation, const Tensor& rotation_t, const Tensor& centroids, const OptTensor& signs,
                      const OptTensor& query_rot, const OptTensor& partial_stats, const OptTensor& partial_values,
                      int64_t bits, int64_t value_group, double scaling, int64_t block_size, bool tq_keys, uintptr_t stream) {
  const at::Device dev = q.device();
  const int dt = dtype_code(q);
  if (!dev.is_cuda() || dt < 0 || !plain(q, dev) || (q.dim() != 3 && q.dim() != 4)) return std::nullopt;
  for (const Tensor* t : {&rk, &rv, &seq_lengths, &rotation, &rotation_t, &centroids})
    if (!plain(*t, dev)) return std::nullopt;
  for (const OptTensor* t : {&gate, &out_in, &key, &key_norms, &vdata, &vscales, &vzeros, &signs, &query_rot,
                             &partial_stats, &partial_values})
    if (!plain(*t, dev)) return std::nullopt;
  const int64_t B = q.size(0), hq = q.size(1), D = q.size(-1);
  if (q.dim() == 4 && q.size(2) != 1) return std::nullopt;
  if (gate && (gate->sizes() != q.sizes() || gate->scalar_type() != q.scalar_type())) return std::nullopt;
  if (rk.dim() != 4 || rv.dim() != 4 || rk.size(0) != B || rk.size(3) != D || rv.sizes() != rk.sizes() ||
      rk.scalar_type() != q.scalar_type() || rv.scalar_type() != q.scalar_type())
    return std::nullopt;
  const int64_t H = rk.size(1);
  if (H < 1 || hq % H != 0 || value_group <= 0 || D % value_group != 0) return std::nullopt;
  if (seq_lengths.scalar_type() != at::kInt || seq_lengths.numel() != B || !seq_lengths.is_contiguous()) return std::nullopt;
  const int64_t per = bits == 2 ? 4 : 2;
  const int64_t C = vdata ? vdata->size(2) : 0;
  if (C > 0) {
    if (!key || !vscales || !vzeros || (tq_keys && !key_norms)) return std::nullopt;
    auto rows = [&](const Tensor& t, int64_t last) {
      return t.dim() == 4 && t.size(0) == B && t.size(1) == H && t.size(2) == C && t.size(3) == last;
    };
    if (!rows(*vdata, D / per) || vdata->scalar_type() != at::kByte || !rows(*vscales, D / value_group) ||
        !rows(*vzeros, D / value_group) || vscales->scalar_type() != q.scalar_type() ||
        vzeros->scalar_type() != q.scalar_type())
      return std::nullopt;
    if (tq_keys ? (!rows(*key, D / per) || key->scalar_type() != at::kByte || key_norms->scalar_type() != at::kHalf ||
                   key_norms->dim() != 3 || key_norms->size(0) != B || key_norms->size(1) != H || key_norms->size(2) != C)
                : (!rows(*key, D) || key->scalar_type() != q.scalar_type()))
      return std::nullopt;
  }
  const bool own = !query_rot;
  if (own != !partial_stats || own != !partial_values) return std::nullopt;
  if (!own && (partial_stats->scalar_type() != at::kFloat || partial_values->scalar_type() != at::kFloat ||
               query_rot->scalar_type() != at::kFloat || query_rot->numel() < B * hq * D || !query_rot->is_contiguous() ||
               partial_stats->dim() != 4 || partial_values->dim() != 4 || partial_stats->size(0) != B ||
               partial_stats->size(1) != hq || partial_values->size(0) != B || partial_values->size(1) != hq ||
               partial_values->size(3) != D))
    return std::nullopt;
  if (signs && (signs->scalar_type() != at::kFloat || signs->numel() != D)) return std::nullopt;
  if (out_in && (out_in->sizes() != q.sizes() || out_in->scalar_type() != q.scalar_type())) return std::nullopt;

  anna_mi_decode_args a{};
  a.dtype = dt;
  a.batch = B, a.q_heads = hq, a.kv_heads = H, a.head_dim = D;
  a.query = query_view(q);
  a.len1 = C;
  a.key_format = tq_keys ? 1 : 0;
  a.value_format = 1;
  if (C > 0) {
    a.key = view(*key);
    if (tq_keys) a.key_norms = view(*key_norms, true);
    a.value = view(*vdata);
    a.value_scales = view(*vscales);
    a.value_zeros = view(*vzeros);
  }
  a.key_bits = a.value_bits = (int)bits;
  a.value_group_size = value_group;
  a.rotation = (const float*)ptr(rotation);
  a.rotation_t = (const float*)ptr(rotation_t);
  a.key_centroids = (const float*)ptr(centroids);
  a.rotation_signs = (const float*)ptr(signs);
  a.len2 = rk.size(2);
  a.residual_key = view(rk);
  a.residual_value = view(rv);
  a.scaling = (float)scaling;
  a.block_size = block_size;
  a.seq_lengths = (const int32_t*)ptr(seq_lengths);
  const int64_t nblk = lib.decode_num_blocks(&a);
  Tensor ws;
  if (own) {
    ws = at::empty({B * hq * (D + nblk * (2 + D))}, q.options().dtype(at::kFloat).requires_grad(false));
    float* const w0 = (float*)ptr(ws);
    a.query_rot = w0;
    a.partial_values = {w0 + B * hq * D, hq * nblk * D, nblk * D, D, 1};
    a.partial_stats = {w0 + B * hq * D * (1 + nblk), hq * nblk * 2, nblk * 2, 2, 1};
    a.partial_capacity = nblk;
  } else {
    a.query_rot = (float*)ptr(query_rot);
    a.partial_stats = view(*partial_stats);
    a.partial_values = view(*partial_values);
    a.partial_capacity = std::min(partial_stats->size(2), partial_values->size(2));
    if (nblk > a.partial_capacity) return std::nullopt;
  }
  Tensor out = out_in ? *out_in : at::empty(q.sizes(), q.options().requires_grad(false));
  a.out = query_view(out);
  if (gate) {
    a.gate_layout = 2;
    a.gate = query_view(*gate);
  }
  check(lib.gqa_decode_splitkv(&a, stream_ptr(stream)), "anna_mi_gqa_decode_splitkv");
  return out;
}

// ---------------------------------------------------------------- 2-bit pool decode

// TurboQuantBatchCache.decode: contiguous bf16 [B, Hq, 256] query (and gate), the cache's own buffers.
OptTensor decode_pool(const Tensor& q, const OptTensor& gate, const OptTensor& out_in, const Tensor& key_codes,
                      const Tensor& key_norms, const Tensor& value_codes, const Tensor& value_norms, const Tensor& rk,
                      const Tensor& rvt, const Tensor& seq_offsets, const Tensor& seq_lengths, const Tensor& signs,
                      const Tensor& partial_stats, const Tensor& partial_values, const Tensor& item_table,
                      int64_t pool_tokens, int64_t window, int64_t kv_heads, int64_t q_heads, int64_t batch,
                      int64_t blocks_per_item, int64_t num_workgroups, double key_scale, double value_scale,
                      double scaling, uintptr_t stream) {
  const at::Device dev = key_codes.device();
  if (!dev.is_cuda() || !is(q, dev, at::kBFloat16) || q.dim() != 3 || q.size(0) != batch || q.size(1) != q_heads ||
      q.size(2) != 256)
    return std::nullopt;
  if (gate && (!is(*gate, dev, at::kBFloat16) || gate->sizes() != q.sizes())) return std::nullopt;
  if (out_in && (!is(*out_in, dev, at::kBFloat16) || out_in->sizes() != q.sizes())) return std::nullopt;
  for (const Tensor* t : {&key_codes, &key_norms, &value_codes, &value_norms, &rk, &rvt, &seq_offsets, &seq_lengths, &signs,
                          &partial_stats, &partial_values, &item_table})
    if (!plain(*t, dev) || !t->is_contiguous()) return std::nullopt;
  Tensor out = out_in ? *out_in : at::empty(q.sizes(), q.options().requires_grad(false));
  anna_mi_tq_decode_args a{};
  a.batch = batch, a.q_heads = q_heads, a.kv_heads = kv_heads, a.head_dim = 256;
  a.key_bits = a.value_bits = 2;
  a.query = (const uint16_t*)ptr(q);
  a.gate = (const uint16_t*)ptr(gate);
  a.key_codes = (const uint8_t*)ptr(key_codes);
  a.key_norms = (const uint16_t*)ptr(key_norms);
  a.value_codes = (const uint8_t*)ptr(value_codes);
  a.value_norms = (const uint16_t*)ptr(value_norms);
  a.pool_tokens = pool_tokens;
  a.residual_key = (const uint16_t*)ptr(rk);
  a.residual_value_t = (const uint16_t*)ptr(rvt);
  a.residual_capacity = window;
  a.seq_offsets = (const int32_t*)ptr(seq_offsets);
  a.seq_lengths = (const int32_t*)ptr(seq_lengths);
  a.signs = (const float*)ptr(signs);
  a.key_scale = (float)key_scale, a.value_scale = (float)value_scale, a.scaling = (float)scaling;
  a.blocks_per_item = blocks_per_item;
  a.num_workgroups = num_workgroups;
  a.partial_stats = (float*)ptr(partial_stats);
  a.partial_values = (float*)ptr(partial_values);
  a.item_table = (int32_t*)ptr(item_table);
  a.out = (uint16_t*)ptr(out);
  check(lib.tq_decode(&a, stream_ptr(stream)), "anna_mi_tq_decode");
  return out;
}

// ---------------------------------------------------------------- one-launch append

// anna_mi_tq_store into slab tensors of one layer; key_signs etc. only for inner-product keys.  Returns
// the lengths before (int64 [batch]).
OptTensor tq_store(const Tensor& k, const Tensor& v, const OptTensor& key_codes, const OptTensor& key_norms,
                   const OptTensor& key_signs, const OptTensor& key_residual_norms, const OptTensor& key_dense,
                   const OptTensor& vdata, const OptTensor& vscales, const OptTensor& vzeros, const Tensor& rk,
                   const Tensor& rv, const Tensor& seq_in, const Tensor& seq_out, const Tensor& seq_lengths,
                   const Tensor& signs,
                   const Tensor& thresholds, const OptTensor& centroids, const OptTensor& gaussian,
                   const OptTensor& gaussian_t, bool ip, int64_t row0, int64_t capacity, int64_t bits,
                   int64_t value_group, int64_t max_leaving, int64_t max_fill, uintptr_t stream) {
  const at::Device dev = rk.device();
  const int dt = dtype_code(rk);
  if (!dev.is_cuda() || dt < 0) return std::nullopt;
  const int64_t per = 16 / (int64_t)rk.element_size();
  for (const Tensor* t : {&k, &v}) {
    if (!plain(*t, dev) || t->dim() != 4 || t->scalar_type() != rk.scalar_type() || t->stride(3) != 1 ||
        t->stride(0) % per || t->stride(1) % per || t->stride(2) % per || (uintptr_t)ptr(*t) % 16 || t->size(2) == 0)
      return std::nullopt;
  }
  if (k.sizes() != v.sizes() || rk.dim() != 4 || k.size(1) != rk.size(1) || k.size(3) != rk.size(3) ||
      row0 < 0 || row0 + k.size(0) > rk.size(0) || !plain(rk, dev) || !plain(rv, dev) || !rk.is_contiguous() ||
      !rv.is_contiguous())
    return std::nullopt;
  for (const Tensor* t : {&seq_in, &seq_out, &seq_lengths, &signs, &thresholds})
    if (!plain(*t, dev) || !t->is_contiguous()) return std::nullopt;
  for (const OptTensor* t : {&key_codes, &key_norms, &key_signs, &key_residual_norms, &key_dense, &vdata, &vscales, &vzeros,
                             &centroids, &gaussian, &gaussian_t})
    if (*t && (!plain(**t, dev) || !(*t)->is_contiguous())) return std::nullopt;
  const int64_t batch = rk.size(0);
  Tensor past = at::empty({batch}, k.options().dtype(at::kLong).requires_grad(false));
  anna_mi_tq_store_args a{};
  a.dtype = dt, a.key_format = ip ? 1 : 0;
  a.batch = batch, a.row0 = row0, a.rows = k.size(0);
  a.kv_heads = k.size(1), a.head_dim = k.size(3), a.tokens = k.size(2);
  a.capacity = capacity, a.residual_capacity = rk.size(2);
  a.key_bits = a.value_bits = (int)bits;
  a.value_group_size = value_group;
  a.new_key = ptr(k), a.new_value = ptr(v);
  a.key_stride_row = k.stride(0), a.key_stride_head = k.stride(1), a.key_stride_token = k.stride(2);
  a.value_stride_row = v.stride(0), a.value_stride_head = v.stride(1), a.value_stride_token = v.stride(2);
  a.key_codes = (uint8_t*)ptr(key_codes);
  a.key_norms = ptr(key_norms);
  a.key_signs = (uint8_t*)ptr(key_signs);
  a.key_residual_norms = (float*)ptr(key_residual_norms);
  a.key_dense = ptr(key_dense);
  a.value_data = (uint8_t*)ptr(vdata);
  a.value_scales = ptr(vscales);
  a.value_zeros = ptr(vzeros);
  a.residual_key = ptr(rk), a.residual_value = ptr(rv);
  a.seq_in = (const int32_t*)ptr(seq_in);
  a.seq_out = (int32_t*)ptr(seq_out);
  a.seq_lengths = (int32_t*)ptr(seq_lengths);
  a.past_out = (int64_t*)ptr(past);
  a.max_leaving = max_leaving, a.max_fill = max_fill;
  a.signs = (const float*)ptr(signs);
  a.thresholds = (const float*)ptr(thresholds);
  a.centroids = (const float*)ptr(centroids);
  a.gaussian = (const float*)ptr(gaussian);
  a.gaussian_t = (const float*)ptr(gaussian_t);
  check(lib.tq_store(&a, stream_ptr(stream)), "anna_mi_tq_store");
  return past;
}

// ---------------------------------------------------------------- sparse MoE block

// Pieces of one workspace tensor, 256-byte aligned
struct Carve {
  size_t used = 0;
  size_t take(size_t bytes) {
    const size_t at = used;
    used += (bytes + 255) & ~size_t(255);
    return at;
  }
};

// The launches of SparseMoeInt4.forward (see anna_amd/moe.py) over one workspace allocation.
OptTensor moe_block(const Tensor& x, const Tensor& logits, const Tensor& gq, const Tensor& gs, const Tensor& gz,
                    const Tensor& uq, const Tensor& us, const Tensor& uz, const Tensor& dq, const Tensor& ds,
                    const Tensor& dz, const Tensor& experts, const Tensor& slots, int64_t group, int64_t top_k,
                    bool normalize, bool small, int64_t max_routes_hint, uintptr_t stream) {
  const at::Device dev = x.device();
  if (!dev.is_cuda() || !plain(x, dev) || !plain(logits, dev) || x.dim() != 2 || logits.dim() != 2) return std::nullopt;
  const int dt = dtype_code(x), ldt = dtype_code(logits), sdt = dtype_code(gs);
  if (dt < 0 || ldt < 0 || sdt < 0 || x.stride(1) != 1 || logits.stride(1) != 1) return std::nullopt;
  const int64_t T = x.size(0), H = x.size(1), E = logits.size(1), R = T * top_k;
  if (T < 1 || logits.size(0) != T || top_k < 1 || top_k > E || x.stride(0) < H || logits.stride(0) < E) return std::nullopt;
  for (const Tensor* t : {&gq, &uq, &dq})
    if (!is(*t, dev, at::kInt) || t->dim() != 3) return std::nullopt;
  for (const Tensor* t : {&gz, &uz, &dz})
    if (!is(*t, dev, at::kChar) || t->dim() != 3) return std::nullopt;
  for (const Tensor* t : {&gs, &us, &ds})
    if (!is(*t, dev, gs.scalar_type()) || t->dim() != 3) return std::nullopt;
  if (gq.sizes() != uq.sizes() || gs.sizes() != us.sizes()) return std::nullopt;
  if (!is(experts, dev, at::kLong) || !is(slots, dev, at::kLong) || experts.numel() != E || slots.numel() != E)
    return std::nullopt;
  const int64_t I = gq.size(1);
  if (dq.size(1) == H && ds.size(2) == H && gs.size(2) == I) {
    anna_mi_moe_prefill_args p{};
    p.dtype = dt, p.logits_dtype = ldt, p.scale_dtype = sdt, p.normalize = normalize;
    p.tokens = T, p.num_experts = E, p.top_k = top_k, p.hidden_dim = H, p.intermediate_dim = I, p.group_size = group;
    p.hidden = ptr(x), p.hidden_row_stride = T > 1 ? x.stride(0) : std::max(H, x.stride(0));
    p.logits = ptr(logits), p.logits_row_stride = logits.stride(0);
    p.slots = (const int64_t*)ptr(slots);
    p.gate_qweight = (const int32_t*)ptr(gq), p.gate_qscale = ptr(gs), p.gate_qzeros = (const int8_t*)ptr(gz);
    p.up_qweight = (const int32_t*)ptr(uq), p.up_qscale = ptr(us), p.up_qzeros = (const int8_t*)ptr(uz);
    p.down_qweight = (const int32_t*)ptr(dq), p.down_qscale = ptr(ds), p.down_qzeros = (const int8_t*)ptr(dz);
    p.hidden_packed_cols = gq.size(2), p.hidden_groups = gs.size(1);
    p.intermediate_packed_cols = dq.size(2), p.intermediate_groups = ds.size(1);
    if (const int64_t bytes = lib.moe_prefill_workspace(&p); bytes > 0) {
      Tensor ws = at::empty({bytes}, x.options().dtype(at::kByte).requires_grad(false));
      Tensor out = at::empty({T, H}, x.options().requires_grad(false));
      p.workspace = ptr(ws), p.out = ptr(out);
      check(lib.moe_prefill(&p, stream_ptr(stream)), "anna_mi_moe_prefill");
      return out;
    }
  }
  const size_t es = (size_t)x.element_size();
  Carve c;
  const size_t o_w = c.take(R * 4), o_sel = c.take(R * 8), o_usage = c.take(E * 4), o_off = c.take((E + 1) * 8),
               o_tok = c.take(R * 8), o_route = c.take(R * 8), o_pos = c.take(R * 8), o_items = c.take((4 + 4 * E) * 4),
               o_cw = c.take(R * es), o_x = c.take(R * H * es), o_y = c.take(R * H * es), o_act = c.take(R * I * 4);
  Tensor ws = at::empty({(int64_t)c.used}, x.options().dtype(at::kByte).requires_grad(false));
  Tensor out = at::empty({T, H}, x.options().requires_grad(false));
  char* const w0 = (char*)ptr(ws);
  float* const w = (float*)(w0 + o_w);
  int64_t *const sel = (int64_t*)(w0 + o_sel), *const off = (int64_t*)(w0 + o_off), *const tok = (int64_t*)(w0 + o_tok),
                 *const route = (int64_t*)(w0 + o_route), *const pos = (int64_t*)(w0 + o_pos);
  int32_t *const usage = (int32_t*)(w0 + o_usage), *const items = (int32_t*)(w0 + o_items);
  void* const st = stream_ptr(stream);
  if (small) {
    check(lib.moe_route_small(ptr(logits), ldt, T, E, logits.stride(0), top_k, normalize, w, sel, usage, off, tok, route, pos,
                              (const int64_t*)ptr(slots), items, st),
          "anna_mi_moe_route_small");
    check(lib.moe_gather(ptr(x), dt, H, x.stride(0), w, ANNA_MI_F32, route, R, top_k, w0 + o_x, w0 + o_cw, st),
          "anna_mi_moe_gather");
  } else {
    check(lib.moe_router(ptr(logits), ldt, T, E, logits.stride(0), top_k, normalize, w, sel, usage, st),
          "anna_mi_moe_router");
    check(lib.moe_dispatch(ptr(x), dt, T, H, x.stride(0), w, ANNA_MI_F32, sel, usage, 0, E, top_k, tok, route, off, w0 + o_x,
                           w0 + o_cw, pos, (const int64_t*)ptr(slots), items, st),
          "anna_mi_moe_dispatch");
  }
  anna_mi_moe_mlp_args a{};
  a.dtype = dt, a.scale_dtype = sdt;
  a.routes = R, a.hidden_dim = H, a.intermediate_dim = I;
  a.compact_hidden = w0 + o_x, a.compact_weights = w0 + o_cw, a.compact_outputs = w0 + o_y;
  a.expert_offsets = off;
  a.active_experts = (const int64_t*)ptr(experts), a.active_slots = (const int64_t*)ptr(slots), a.active_count = E;
  a.gate_qweight = (const int32_t*)ptr(gq), a.gate_qscale = ptr(gs), a.gate_qzeros = (const int8_t*)ptr(gz);
  a.up_qweight = (const int32_t*)ptr(uq), a.up_qscale = ptr(us), a.up_qzeros = (const int8_t*)ptr(uz);
  a.down_qweight = (const int32_t*)ptr(dq), a.down_qscale = ptr(ds), a.down_qzeros = (const int8_t*)ptr(dz);
  a.hidden_packed_cols = gq.size(2), a.hidden_groups = gs.size(1);
  a.intermediate_packed_cols = dq.size(2), a.intermediate_groups = ds.size(1);
  a.group_size = group;
  a.activation = (float*)(w0 + o_act);
  a.sweep_chunks = (int)std::min<int64_t>(4, std::max<int64_t>(1, (max_routes_hint + 15) / 16));
  a.items = items, a.items_prefilled = 1;
  check(lib.moe_grouped_int4_mlp(&a, st), "anna_mi_moe_grouped_int4_mlp");
  check(lib.moe_combine(w0 + o_y, dt, H, pos, T, top_k, ptr(out), st), "anna_mi_moe_combine");
  return out;
}

// ---------------------------------------------------------------- paged cache

anna_mi_paged* paged(uintptr_t handle) { return reinterpret_cast<anna_mi_paged*>(handle); }
anna_mi_paged_span* span_at(uintptr_t address) { return reinterpret_cast<anna_mi_paged_span*>(address); }

// Whole numbers of a list or tuple, each within [low, high]; nullopt for anything else.
template <class T> std::optional<std::vector<T>> whole(const py::handle& list, int64_t low, int64_t high) {
  if (!PyList_CheckExact(list.ptr()) && !PyTuple_CheckExact(list.ptr())) return std::nullopt;
  PyObject** items = PySequence_Fast_ITEMS(list.ptr());
  std::vector<T> v(PySequence_Fast_GET_SIZE(list.ptr()));
  for (size_t i = 0; i < v.size(); i++) {
    if (!PyLong_CheckExact(items[i])) return std::nullopt;
    int overflow = 0;
    const long long x = PyLong_AsLongLongAndOverflow(items[i], &overflow);
    if (overflow || x < low || x > high) return std::nullopt;
    v[i] = (T)x;
  }
  return v;
}
constexpr int64_t I32 = INT32_MAX, I64 = INT64_MAX / 4;

py::object paged_fork(uintptr_t handle, const py::object& parents, uintptr_t stream) {
  const auto p = whole<int32_t>(parents, 0, I32);
  if (!p) return py::none();
  std::vector<int32_t> children(p->size());
  check(lib.paged_fork(paged(handle), (int64_t)p->size(), p->data(), children.data(), stream_ptr(stream)), "anna_mi_paged_fork");
  return py::cast(children);
}

bool paged_free(uintptr_t handle, const py::object& seqs, uintptr_t stream) {
  const auto s = whole<int32_t>(seqs, 0, I32);
  if (!s) return false;
  check(lib.paged_free(paged(handle), (int64_t)s->size(), s->data(), stream_ptr(stream)), "anna_mi_paged_free");
  return true;
}

// A span's memory, and the span's pointers to it; starts null: of an extend by counts.
std::vector<Tensor> span_memory(uintptr_t handle, anna_mi_paged_span* out, const std::vector<int32_t>& s, const int64_t* starts,
                                const std::vector<int64_t>& counts, int64_t kv_heads, int64_t head_dim, int64_t device) {
  check(lib.paged_span_plan(paged(handle), (int64_t)s.size(), s.data(), starts, counts.data(), out), "anna_mi_paged_span_plan");
  const auto ints = at::TensorOptions().dtype(at::kInt).device(at::kCUDA, (c10::DeviceIndex)device);
  std::vector<Tensor> held{at::empty({out->words}, ints)};
  if (out->partial_rows > 0) {
    held.push_back(at::empty({out->partial_rows, kv_heads, 2}, ints.dtype(at::kFloat)));
    held.push_back(at::empty({out->partial_rows, kv_heads, head_dim}, ints.dtype(at::kFloat)));
    out->partial_stats = (float*)ptr(held[1]);
    out->partial_values = (float*)ptr(held[2]);
  }
  out->buf = (int32_t*)ptr(held[0]);
  return held;
}

// Fills a span anew, with its buffer and workspace: extend (starts is None) by counts, None for one each, or the
// tokens that the sequences hold already.  -> (seqs, starts, counts, tensors), or None.
py::object paged_span(uintptr_t handle, uintptr_t span, const py::object& seqs, const py::object& starts, const py::object& counts,
                      int64_t max_length, int64_t kv_heads, int64_t head_dim, int64_t device, uintptr_t stream) {
  const auto s = whole<int32_t>(seqs, 0, I32);
  if (!s) return py::none();
  const int64_t n = (int64_t)s->size();
  anna_mi_paged_span* out = span_at(span);
  std::optional<std::vector<int64_t>> c, at;
  std::vector<Tensor> held;
  if (counts.is_none()) c = std::vector<int64_t>(n, 1);
  else c = whole<int64_t>(counts, 0, I64);
  if (!c || (int64_t)c->size() != n) return py::none();
  if (starts.is_none()) {
    at = std::vector<int64_t>(n);
    check(lib.paged_lengths(paged(handle), n, s->data(), at->data(), nullptr), "anna_mi_paged_lengths");
    for (int64_t i = 0; i < n; i++)
      if ((*at)[i] < 0 || (*c)[i] > max_length - (*at)[i]) return py::none();
    held = span_memory(handle, out, *s, nullptr, *c, kv_heads, head_dim, device);  // before anything changes
    check(lib.paged_extend(paged(handle), n, s->data(), c->data(), at->data(), stream_ptr(stream)), "anna_mi_paged_extend");
  } else {
    at = whole<int64_t>(starts, 0, I64);
    if (!at || (int64_t)at->size() != n) return py::none();
    held = span_memory(handle, out, *s, at->data(), *c, kv_heads, head_dim, device);
  }
  check(lib.paged_span_fill(paged(handle), n, s->data(), at->data(), c->data(), out, stream_ptr(stream)), "anna_mi_paged_span_fill");
  return py::make_tuple(*s, *at, *c, held);
}

// Rows [tokens, heads, head_dim] of the cache's type that the kernels read as they are
bool paged_rows(const Tensor& t, const at::Device& dev, at::ScalarType dt, int64_t tokens, int64_t heads, int64_t head_dim) {
  return plain(t, dev) && !(t.requires_grad() && at::GradMode::is_enabled()) && t.scalar_type() == dt && t.dim() == 3 && t.size(0) == tokens && t.size(1) == heads && t.size(2) == head_dim &&
         t.stride(2) == 1 && (tokens <= 1 || t.stride(0) % 8 == 0) && (heads <= 1 || t.stride(1) % 8 == 0) &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
int64_t token_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : 0; }
int64_t head_stride(const Tensor& t) { return t.size(1) > 1 ? t.stride(1) : 0; }

bool paged_store(uintptr_t handle, int64_t layer, uintptr_t span, const Tensor& keys, const Tensor& values, const Tensor& pool,
                 at::ScalarType dtype, int64_t head_dim, bool capturing, uintptr_t stream) {
  anna_mi_paged_span* s = span_at(span);
  if (!paged_rows(keys, pool.device(), dtype, s->tokens, pool.size(2), head_dim) ||
      !paged_rows(values, pool.device(), dtype, s->tokens, pool.size(2), head_dim))
    return false;
  check(lib.paged_store(paged(handle), layer, s, ptr(keys), token_stride(keys), head_stride(keys), ptr(values), token_stride(values),
                        head_stride(values), capturing, stream_ptr(stream)),
        "anna_mi_paged_store");
  return true;
}

std::pair<Tensor, Tensor> paged_read(uintptr_t handle, int64_t layer, uintptr_t span, const Tensor& pool, at::ScalarType dtype,
                                     int64_t head_dim, bool capturing, uintptr_t stream) {
  const anna_mi_paged_span* s = span_at(span);
  Tensor keys = at::empty({s->tokens, pool.size(2), head_dim}, pool.options().dtype(dtype)), values = at::empty_like(keys);
  check(lib.paged_read(paged(handle), layer, s, ptr(keys), ptr(values), capturing, stream_ptr(stream)), "anna_mi_paged_read");
  return {keys, values};
}

OptTensor paged_attend(uintptr_t handle, int64_t layer, uintptr_t span, const Tensor& query, const OptTensor& gate, const OptTensor& out,
                       const Tensor& pool, at::ScalarType dtype, int64_t q_heads, int64_t head_dim, double scaling, bool capturing,
                       uintptr_t stream) {
  const anna_mi_paged_span* s = span_at(span);
  const at::Device dev = pool.device();
  if (!paged_rows(query, dev, dtype, s->tokens, q_heads, head_dim) || (gate && !paged_rows(*gate, dev, dtype, s->tokens, q_heads, head_dim)) ||
      (out && (!paged_rows(*out, dev, dtype, s->tokens, q_heads, head_dim) || !out->is_contiguous())) || !(scaling > 0.0 && scaling < 1e30))
    return std::nullopt;
  Tensor o = out ? *out : at::empty({s->tokens, q_heads, head_dim}, query.options().requires_grad(false));
  check(lib.paged_attend(paged(handle), layer, s, ptr(query), token_stride(query), head_stride(query), ptr(gate),
                         gate ? token_stride(*gate) : 0, gate ? head_stride(*gate) : 0, ptr(o), (float)scaling, capturing,
                         stream_ptr(stream)),
        "anna_mi_paged_attend");
  return o;
}

// ---------------------------------------------------------------- linear attention

// Without a gradient or a tangent to lose
bool given(const Tensor& t, const at::Device& dev) {
  return plain(t, dev) && !(t.requires_grad() && at::GradMode::is_enabled()) && !t._fw_grad(0).defined();
}
bool given(const OptTensor& t, const at::Device& dev) { return !t || given(*t, dev); }
// What a call has written, so that autograd sees it where it keeps the tensor; inference tensors have no version
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A pool of states [slots][shape], contiguous in each slot; -> elements from one slot to the next, or -1
int64_t pool_stride(const Tensor& t, const at::Device& dev, at::ScalarType dt, at::IntArrayRef shape) {
  if (!given(t, dev) || t.scalar_type() != dt || t.dim() != (int64_t)shape.size() + 1) return -1;
  int64_t size = 1;
  for (int64_t i = (int64_t)shape.size(); i > 0; i--) {
    if (t.size(i) != shape[i - 1] || (t.size(i) > 1 && t.stride(i) != size)) return -1;
    size *= t.size(i);
  }
  return t.size(0) > 1 ? (t.stride(0) >= size ? t.stride(0) : -1) : size;
}

// Bytes that a tensor's elements lie in, and whether those of two may meet
std::pair<intptr_t, intptr_t> memory(const Tensor& t) {
  const intptr_t start = reinterpret_cast<intptr_t>(ptr(t));
  if (t.numel() == 0) return {start, start};
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); i++) last += (t.size(i) - 1) * t.stride(i);
  return {start, start + (last + 1) * (int64_t)t.element_size()};
}
bool may_meet(const Tensor& state, std::initializer_list<const Tensor*> inputs) {
  const auto [low, high] = memory(state);
  for (const Tensor* t : inputs) {
    if (!t) continue;
    const auto [first, end] = memory(*t);
    if (first < high && low < end) return true;
  }
  return false;
}
const Tensor* of(const OptTensor& t) { return t ? &*t : nullptr; }

OptTensor gated_delta(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& decay, const Tensor& beta,
                      const Tensor& state, const OptTensor& a_log, const OptTensor& dt_bias, uintptr_t span_address, int64_t device,
                      double scaling, bool normalize, uintptr_t stream) {
  auto* span = reinterpret_cast<anna_mi_state_span*>(span_address);
  const at::Device dev = query.device();
  const at::ScalarType dt = query.scalar_type();
  if (!query.is_cuda() || dev.index() != device || query.dim() != 3 || value.dim() != 3 || (dt != at::kBFloat16 && dt != at::kHalf) || span->tokens != query.size(0)) return std::nullopt;
  const int64_t tokens = query.size(0), HK = query.size(1), DK = query.size(2), HV = value.size(1), DV = value.size(2);
  auto lies = [&](const Tensor& t, int64_t heads, int64_t dim) { return given(t, dev) && paged_rows(t, dev, dt, tokens, heads, dim); };
  if (!lies(query, HK, DK) || !lies(key, HK, DK) || !lies(value, HV, DV))
    return std::nullopt;
  auto rows = [&](const Tensor& t) {
    return given(t, dev) && t.scalar_type() == decay.scalar_type() && dtype_code(t) >= 0 && t.dim() == 2 && t.size(0) == tokens &&
           t.size(1) == HV && (t.stride(1) == 1 || HV == 1);
  };
  auto heads = [&](const OptTensor& t) { return !t || (given(*t, dev) && is(*t, dev, at::kFloat) && t->dim() == 1 && t->size(0) == HV); };
  if (!rows(decay) || !rows(beta) || a_log.has_value() != dt_bias.has_value() || !heads(a_log) || !heads(dt_bias) ||
      (DK != 64 && DK != 128) || DV % 32 || DV < 32 || DV > 256 || HK < 1 || HV < 1 || HV % HK || !(scaling > -1e30 && scaling < 1e30))
    return std::nullopt;
  const int64_t stride = pool_stride(state, dev, at::kFloat, {HV, DK, DV});
  if (stride < 0 || stride % 4 || reinterpret_cast<uintptr_t>(ptr(state)) % 16 ||
      may_meet(state, {&query, &key, &value, &decay, &beta, of(a_log), of(dt_bias)}))
    return std::nullopt;
  Tensor out = at::empty({tokens, HV, DV}, value.options().requires_grad(false)), workspace;
  anna_mi_gated_delta_args a{};
  a.dtype = dtype_code(query), a.gates_dtype = dtype_code(decay), a.normalize = normalize, a.scaling = (float)scaling;
  a.key_heads = HK, a.value_heads = HV, a.key_dim = DK, a.value_dim = DV;
  a.query = ptr(query), a.query_stride_token = token_stride(query), a.query_stride_head = head_stride(query);
  a.key = ptr(key), a.key_stride_token = token_stride(key), a.key_stride_head = head_stride(key);
  a.value = ptr(value), a.value_stride_token = token_stride(value), a.value_stride_head = head_stride(value);
  a.decay = ptr(decay), a.decay_stride = token_stride(decay), a.beta = ptr(beta), a.beta_stride = token_stride(beta);
  a.a_log = (const float*)ptr(a_log), a.dt_bias = (const float*)ptr(dt_bias);
  a.state = (float*)ptr(state), a.slots = state.size(0), a.state_stride_slot = stride, a.out = ptr(out);
  if (span->chunks > 0) {
    workspace = at::empty({lib.gated_delta_workspace(&a, span)}, value.options().dtype(at::kByte).requires_grad(false));
    a.workspace = ptr(workspace);
  }
  check(lib.gated_delta(&a, span, stream_ptr(stream)), "anna_mi_gated_delta");
  written(state);
  return out;
}

OptTensor causal_conv1d(const Tensor& x, const Tensor& weight, const OptTensor& bias, const Tensor& state, uintptr_t span_address,
                        int64_t device, bool silu, uintptr_t stream) {
  auto* span = reinterpret_cast<anna_mi_state_span*>(span_address);
  const at::Device dev = x.device();
  const at::ScalarType dt = x.scalar_type();
  if (!x.is_cuda() || dev.index() != device || x.dim() != 2 || dtype_code(x) < 0 || !given(x, dev) || span->tokens != x.size(0)) return std::nullopt;
  const int64_t tokens = x.size(0), channels = x.size(1);
  if (channels < 1 || (channels > 1 && x.stride(1) != 1) || (tokens > 1 && x.stride(0) < channels) || !given(weight, dev) ||
      !is(weight, dev, dt) || weight.dim() != 2 || weight.size(0) != channels || weight.size(1) < 2 || weight.size(1) > 8 ||
      !given(bias, dev) || (bias && (!is(*bias, dev, dt) || bias->dim() != 1 || bias->size(0) != channels)))
    return std::nullopt;
  const int64_t width = weight.size(1), stride = pool_stride(state, dev, dt, {width - 1, channels});
  if (stride < 0 || may_meet(state, {&x, &weight, of(bias)})) return std::nullopt;
  Tensor out = at::empty({tokens, channels}, x.options().requires_grad(false));
  check(lib.causal_conv1d(ptr(x), dtype_code(x), channels, tokens > 1 ? x.stride(0) : channels, ptr(weight), width, ptr(bias), ptr(state),
                          state.size(0), stride, silu, span, ptr(out), channels, stream_ptr(stream)),
        "anna_mi_causal_conv1d");
  written(state);
  return out;
}

// Whether rows share no element: of other memory, or other columns of one matrix
bool rows_apart(const Tensor& a, int64_t a_stride, const Tensor& b, int64_t b_stride, int64_t cols) {
  const int64_t size = a.element_size(), between = reinterpret_cast<intptr_t>(ptr(b)) - reinterpret_cast<intptr_t>(ptr(a));
  if (between >= ((a.numel() / cols - 1) * a_stride + cols) * size || -between >= ((b.numel() / cols - 1) * b_stride + cols) * size) return true;
  if (a_stride != b_stride || between % size) return false;
  const int64_t column = (between / size % a_stride + a_stride) % a_stride;
  return column >= cols && column <= a_stride - cols;
}

// out, or with a group codes, and scales; undefined for calls that are left to the caller
Tensor norm(const Tensor& x, const Tensor& weight, double eps, double weight_offset, const OptTensor& residual, const OptTensor& gate,
            int64_t group, Tensor* scales, int64_t device, uintptr_t stream) {
  const Tensor none;
  const at::Device dev = x.device();
  const at::ScalarType dt = x.scalar_type();
  if (!x.is_cuda() || dev.index() != device || x.dim() < 1 || dtype_code(x) < 0 || x.numel() == 0 || !(eps >= 0.0 && eps < 1e30)) return none;
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  // rows with one stride: contiguous tensors, and matrices
  auto lies = [&](const Tensor& t, int64_t& stride) {
    if (!given(t, dev) || t.scalar_type() != dt || t.sizes() != x.sizes()) return false;
    if (t.is_contiguous()) return stride = cols, true;
    if (t.dim() != 2 || (cols > 1 && t.stride(1) != 1) || (rows > 1 && t.stride(0) < cols)) return false;
    return stride = rows > 1 ? t.stride(0) : cols, true;
  };
  anna_mi_rms_norm_args a{};
  if (!lies(x, a.x_stride) || (residual && !lies(*residual, a.residual_stride)) || (gate && !lies(*gate, a.gate_stride)) ||
      !given(weight, dev) || !is(weight, dev, dt) || weight.dim() != 1 || weight.size(0) != cols)
    return none;
  if (residual && ((!(ptr(*residual) == ptr(x) && a.residual_stride == a.x_stride) && !rows_apart(*residual, a.residual_stride, x, a.x_stride, cols)) ||
                   (gate && !rows_apart(*residual, a.residual_stride, *gate, a.gate_stride, cols)) ||
                   !rows_apart(*residual, a.residual_stride, weight, cols, cols)))
    return none;
  a.dtype = dtype_code(x), a.out_format = group > 0, a.rows = rows, a.cols = cols, a.group = group;
  a.x = ptr(x), a.weight = ptr(weight), a.residual = ptr(residual), a.gate = ptr(gate);
  a.eps = (float)eps, a.weight_offset = (float)weight_offset, a.out_stride = cols;
  const auto options = x.options().requires_grad(false);
  Tensor out = at::empty(x.sizes(), group > 0 ? options.dtype(at::kFloat8_e4m3fn) : options);
  a.out = ptr(out);
  if (group > 0) {
    auto shape = x.sizes().vec();
    shape.back() = cols / group;
    *scales = at::empty(shape, options.dtype(at::kFloat));
    a.scales = (float*)ptr(*scales);
  }
  check(lib.rms_norm(&a, stream_ptr(stream)), "anna_mi_rms_norm");
  if (residual) written(*residual);
  return out;
}

OptTensor rms_norm(const Tensor& x, const Tensor& weight, double eps, double weight_offset, const OptTensor& residual, const OptTensor& gate,
                   int64_t device, uintptr_t stream) {
  Tensor out = norm(x, weight, eps, weight_offset, residual, gate, 0, nullptr, device, stream);
  return out.defined() ? OptTensor(std::move(out)) : std::nullopt;
}

std::optional<std::pair<Tensor, Tensor>> rms_norm_e4m3(const Tensor& x, const Tensor& weight, double eps, double weight_offset,
                                                       const OptTensor& residual, const OptTensor& gate, int64_t group, int64_t device,
                                                       uintptr_t stream) {
  Tensor scales, codes = norm(x, weight, eps, weight_offset, residual, gate, group, &scales, device, stream);
  if (!codes.defined()) return std::nullopt;
  return std::make_pair(std::move(codes), std::move(scales));
}

}  // namespace

#ifndef ANNA_MI_SOURCE_HASH
#define ANNA_MI_SOURCE_HASH "unstamped"
#endif

PYBIND11_MODULE(_torch_host, m) {
  const auto no_gil = py::call_guard<py::gil_scoped_release>();
  m.def("source_hash", [] { return std::string(ANNA_MI_SOURCE_HASH); });
  m.def("bind", &bind);
  m.def("int4_linear", &int4_linear, no_gil, py::arg("x"), py::arg("qweight"), py::arg("qscale"), py::arg("qzeros"),
        py::arg("bias"), py::arg("group"), py::arg("out_features"), py::arg("compute"), py::arg("stream"),
        py::arg("strategies") = true);
  m.def("decode_rows", &decode_rows, no_gil);
  m.def("decode_pool", &decode_pool, no_gil);
  m.def("tq_store", &tq_store, no_gil);
  m.def("moe_block", &moe_block, no_gil);
  m.def("paged_fork", &paged_fork);
  m.def("paged_free", &paged_free);
  m.def("paged_span", &paged_span);
  m.def("paged_store", &paged_store, no_gil);
  m.def("paged_read", &paged_read, no_gil);
  m.def("paged_attend", &paged_attend, no_gil);
  m.def("gated_delta", &gated_delta, no_gil);
  m.def("causal_conv1d", &causal_conv1d, no_gil);
  m.def("rms_norm", &rms_norm, no_gil);
  m.def("rms_norm_e4m3", &rms_norm_e4m3, no_gil);
}
