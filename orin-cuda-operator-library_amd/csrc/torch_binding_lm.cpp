// torch.ops.operatorlib.{rope_append, paged_attention, masked_attention} over
// the C ABI (operatorlib/lm_c.h): what torch_binding.cpp is for the other
// operators, with the same checks (torch_operands.hpp), the same error texts'
// form and the same rules for streams, devices and scratch. Strided inputs are
// taken in place where the C ABI takes strides, and never copied.

#include <ATen/ATen.h>
#include <torch/library.h>

#include <cmath>
#include <cstddef>
#include <cstdint>
#include <limits>
#include <optional>
#include <tuple>

#include "operatorlib/lm_c.h"
#include "torch_operands.hpp"

namespace {

using OptTensor = std::optional<at::Tensor>;

const std::int32_t* ints(const at::Tensor& t) { return static_cast<const std::int32_t*>(caddr(t)); }
const std::int32_t* ints(const OptTensor& t) { return t ? ints(*t) : nullptr; }
const float* floats(const OptTensor& t) { return t ? static_cast<const float*>(caddr(*t)) : nullptr; }
const operatorlib_half_t* half_in(const at::Tensor& t) {
  return static_cast<const operatorlib_half_t*>(caddr(t));
}
operatorlib_half_t* half_out(const at::Tensor& t) {
  return t.defined() ? static_cast<operatorlib_half_t*>(t.data_ptr()) : nullptr;
}
const float* float_in(const at::Tensor& t) { return static_cast<const float*>(caddr(t)); }
float* float_out(const at::Tensor& t) {
  return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr;
}

// A stride of a dimension of one element is nobody's: `dense` stands for it.
std::int64_t stride_of(const at::Tensor& t, std::int64_t dim, std::int64_t dense) {
  return t.size(dim) == 1 ? dense : t.stride(dim);
}

// [tokens, heads, dim] whose token rows are contiguous; gives the distance of
// two tokens.
std::int64_t token_rows(const Operands& in, const at::Tensor& t, const char* name) {
  const std::int64_t dim = t.size(2);
  TORCH_CHECK(stride_of(t, 2, 1) == 1 && stride_of(t, 1, dim) == dim, in.op(), ": ", name,
              " must be contiguous within a token (strides ", t.strides(), ")");
  return stride_of(t, 0, t.size(1) * dim);
}

void require_16_byte_rows(const Operands& in, const at::Tensor& t, const char* name,
                          std::int64_t dim) {
  const std::int64_t chunk = in.half() ? 8 : 4;
  TORCH_CHECK(dim % chunk == 0, in.op(), ": head dimension ", dim, " is not a multiple of ", chunk);
  bool ok = reinterpret_cast<std::uintptr_t>(t.data_ptr()) % 16 == 0;
  for (std::int64_t d = 0; d + 1 < t.dim(); ++d) ok = ok && (t.size(d) == 1 || t.stride(d) % chunk == 0);
  TORCH_CHECK(ok, in.op(), ": the rows of ", name, " must be 16-byte aligned (strides ", t.strides(), ")");
}

struct Cache {
  int pages, kv_heads, page_size, dim;
};

Cache cache_sizes(const Operands& in, const at::Tensor& key_cache, const at::Tensor& value_cache) {
  require_rank(in, key_cache, "key_cache", 4, "[pages, kv_heads, page_size, head_dim]");
  TORCH_CHECK(value_cache.sizes() == key_cache.sizes(), in.op(),
              ": key_cache and value_cache must have the same shape, got ", key_cache.sizes(),
              " and ", value_cache.sizes());
  TORCH_CHECK(key_cache.is_contiguous() && value_cache.is_contiguous(), in.op(),
              ": key_cache and value_cache must be contiguous (dense row-major)");
  return {extent(in.op(), "pages", key_cache.size(0)), extent(in.op(), "kv_heads", key_cache.size(1)),
          extent(in.op(), "page size", key_cache.size(2)),
          extent(in.op(), "head dimension", key_cache.size(3))};
}

std::tuple<at::Tensor, at::Tensor> rope_append_op(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& positions,
    const at::Tensor& frequencies, const at::Tensor& slots, const at::Tensor& key_cache,
    const at::Tensor& value_cache, const OptTensor& axes, bool interleaved, bool return_keys) {
  const Operands in("rope_append", kFloat32OrFloat16,
                    {{&q, "q"}, {&k, "k"}, {&v, "v"}, {&key_cache, "key_cache"},
                     {&value_cache, "value_cache"}}, false);
  require_rank(in, q, "q", 3, "[tokens, heads, head_dim]");
  require_rank(in, k, "k", 3, "[tokens, kv_heads, head_dim]");
  TORCH_CHECK(v.sizes() == k.sizes(), "rope_append: k and v must have the same shape, got ",
              k.sizes(), " and ", v.sizes());
  const Cache cache = cache_sizes(in, key_cache, value_cache);
  const int tokens = extent(in.op(), "tokens", q.size(0));
  const int q_heads = extent(in.op(), "heads", q.size(1));
  const int dim = extent(in.op(), "head dimension", q.size(2));
  TORCH_CHECK(k.size(0) == tokens && k.size(1) == cache.kv_heads && k.size(2) == dim &&
                  cache.dim == dim,
              "rope_append: q ", q.sizes(), ", k ", k.sizes(), " and key_cache ",
              key_cache.sizes(), " do not agree in tokens, kv_heads or head dimension");
  TORCH_CHECK(key_cache.data_ptr() != value_cache.data_ptr(),
              "rope_append: key_cache and value_cache must be different tensors");
  require_aux(in, positions, "positions", at::kInt);
  require_aux(in, frequencies, "frequencies", at::kFloat);
  require_aux(in, slots, "slots", at::kInt);
  TORCH_CHECK(slots.dim() == 1 && slots.size(0) == tokens,
              "rope_append: slots must be [tokens], got ", slots.sizes());
  TORCH_CHECK((positions.dim() == 1 || positions.dim() == 2) && positions.size(-1) == tokens &&
                  positions.numel() > 0,
              "rope_append: positions must be [tokens] or [axes, tokens], got ", positions.sizes());
  const int rows = positions.dim() == 2 ? extent(in.op(), "position axes", positions.size(0)) : 1;
  TORCH_CHECK(frequencies.dim() == 1 && 2 * frequencies.size(0) <= dim,
              "rope_append: frequencies must be [rotary_dim / 2] with rotary_dim at most the head "
              "dimension, got ", frequencies.sizes());
  const int rotary = static_cast<int>(2 * frequencies.size(0));
  if (axes) {
    require_aux(in, *axes, "axes", at::kInt);
    TORCH_CHECK(axes->dim() == 1 && axes->size(0) == frequencies.size(0),
                "rope_append: axes must be [rotary_dim / 2], got ", axes->sizes());
  }
  const std::int64_t qs = token_rows(in, q, "q"), ks = token_rows(in, k, "k"),
                     vs = token_rows(in, v, "v");
  at::Tensor q_out = at::empty(q.sizes(), q.options());
  at::Tensor k_out;  // undefined (None) unless asked for
  if (return_keys) k_out = at::empty(k.sizes(), k.options());
  launch(in, [&](void* s) {
    return in.half()
               ? operatorlib_rope_append_f16(
                     half_in(q), qs, half_in(k), ks, half_in(v), vs, ints(positions), rows,
                     ints(axes), float_in(frequencies), ints(slots), half_out(q_out),
                     half_out(k_out), half_out(key_cache), half_out(value_cache), tokens, q_heads,
                     cache.kv_heads, dim, rotary, interleaved, cache.pages, cache.page_size, s)
               : operatorlib_rope_append_f32(
                     float_in(q), qs, float_in(k), ks, float_in(v), vs, ints(positions), rows,
                     ints(axes), float_in(frequencies), ints(slots), float_out(q_out),
                     float_out(k_out), float_out(key_cache), float_out(value_cache), tokens,
                     q_heads, cache.kv_heads, dim, rotary, interleaved, cache.pages,
                     cache.page_size, s);
  });
  return {q_out, k_out};
}

// What both attentions check of their score rules.
float scale_of(const Operands& in, const std::optional<double>& scale, int dim) {
  const float s = scale ? static_cast<float>(*scale) : 1.0f / std::sqrt(static_cast<float>(dim));
  TORCH_CHECK(std::isfinite(s) && s > 0.0f, in.op(), ": scale must be finite and > 0, got ", s);
  return s;
}

float softcap_of(const Operands& in, double softcap) {
  const float c = static_cast<float>(softcap);
  TORCH_CHECK(std::isfinite(c) && c >= 0.0f, in.op(),
              ": softcap must be finite and >= 0 (0: none), got ", softcap);
  return c;
}

int window_of(const Operands& in, std::int64_t window) {
  TORCH_CHECK(window >= 0 && window <= std::numeric_limits<int>::max(), in.op(),
              ": window must be >= 0 (0: none), got ", window);
  return static_cast<int>(window);
}

void check_slopes(const Operands& in, const OptTensor& slopes, int heads) {
  if (!slopes) return;
  require_aux(in, *slopes, "slopes", at::kFloat);
  TORCH_CHECK(slopes->dim() == 1 && slopes->size(0) == heads, in.op(),
              ": slopes must be [heads], got ", slopes->sizes());
}

void check_heads(const Operands& in, int heads, int kv_heads, int dim) {
  TORCH_CHECK(heads % kv_heads == 0, in.op(), ": ", heads, " heads are not a multiple of ",
              kv_heads, " key heads");
  TORCH_CHECK(dim <= 128, in.op(), ": head dimension ", dim, " is not supported (at most 128)");
}

at::Tensor paged_attention_op(const at::Tensor& q, const at::Tensor& key_cache,
                              const at::Tensor& value_cache, const at::Tensor& page_table,
                              const at::Tensor& lengths, std::optional<double> scale,
                              std::int64_t window, double softcap, const OptTensor& slopes) {
  const Operands in("paged_attention", kFloat32OrFloat16,
                    {{&q, "q"}, {&key_cache, "key_cache"}, {&value_cache, "value_cache"}}, false);
  require_rank(in, q, "q", 3, "[batch, heads, head_dim]");
  const Cache cache = cache_sizes(in, key_cache, value_cache);
  const int batch = extent(in.op(), "batch", q.size(0));
  const int heads = extent(in.op(), "heads", q.size(1));
  const int dim = extent(in.op(), "head dimension", q.size(2));
  TORCH_CHECK(dim == cache.dim, "paged_attention: q has head dimension ", dim,
              " but the cache has ", cache.dim);
  check_heads(in, heads, cache.kv_heads, dim);
  TORCH_CHECK(page_table.device() == q.device() && lengths.device() == q.device(),
              "paged_attention: page_table and lengths must be on ", q.device());
  TORCH_CHECK(page_table.scalar_type() == at::kInt && page_table.dim() == 2 &&
                  page_table.size(0) == batch && page_table.size(1) > 0 &&
                  stride_of(page_table, 1, 1) == 1,
              "paged_attention: page_table must be int32 [batch, pages] with contiguous rows, got ",
              page_table.scalar_type(), " ", page_table.sizes());
  const int max_pages = extent(in.op(), "page_table width", page_table.size(1));
  require_aux(in, lengths, "lengths", at::kInt);
  TORCH_CHECK(lengths.dim() == 1 && lengths.size(0) == batch,
              "paged_attention: lengths must be [batch], got ", lengths.sizes());
  check_slopes(in, slopes, heads);
  const float sc = scale_of(in, scale, dim), cap = softcap_of(in, softcap);
  const int win = window_of(in, window);
  const std::int64_t qs = token_rows(in, q, "q");
  require_16_byte_rows(in, q, "q", dim);
  require_16_byte_rows(in, key_cache, "key_cache", dim);
  require_16_byte_rows(in, value_cache, "value_cache", dim);
  const std::int64_t ts = stride_of(page_table, 0, max_pages);
  at::Tensor out = at::empty(q.sizes(), q.options());
  launch(in, [&](void* s) {
    if (in.half()) {
      const Workspace ws(in, operatorlib_paged_attention_f16_workspace_size(
                                 batch, heads, cache.kv_heads, dim, cache.page_size, max_pages));
      return operatorlib_paged_attention_f16_ws(
          half_in(q), qs, half_in(key_cache), half_in(value_cache), ints(page_table), ts,
          ints(lengths), floats(slopes), half_out(out), batch, heads, cache.kv_heads, dim,
          cache.pages, cache.page_size, max_pages, sc, win, cap, ws.data(), ws.bytes(), s);
    }
    const Workspace ws(in, operatorlib_paged_attention_f32_workspace_size(
                               batch, heads, cache.kv_heads, dim, cache.page_size, max_pages));
    return operatorlib_paged_attention_f32_ws(
        float_in(q), qs, float_in(key_cache), float_in(value_cache), ints(page_table), ts,
        ints(lengths), floats(slopes), float_out(out), batch, heads, cache.kv_heads, dim,
        cache.pages, cache.page_size, max_pages, sc, win, cap, ws.data(), ws.bytes(), s);
  });
  return out;
}

operatorlib_strides_t strides_of(const Operands& in, const at::Tensor& t, const char* name) {
  const std::int64_t dim = t.size(3);
  TORCH_CHECK(stride_of(t, 3, 1) == 1, in.op(), ": the head dimension of ", name,
              " must be contiguous (strides ", t.strides(), ")");
  require_16_byte_rows(in, t, name, dim);
  TORCH_CHECK(stride_of(t, 2, dim) >= dim, in.op(), ": the tokens of ", name,
              " overlap (strides ", t.strides(), ")");
  return {stride_of(t, 0, 0), stride_of(t, 1, 0), stride_of(t, 2, dim)};
}

at::Tensor masked_attention_op(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               bool causal, std::int64_t window, double softcap,
                               const OptTensor& slopes, const OptTensor& documents,
                               const OptTensor& prefixes, std::optional<double> scale) {
  const Operands in("masked_attention", kFloat32OrFloat16, {{&q, "q"}, {&k, "k"}, {&v, "v"}},
                    false);
  require_rank(in, q, "q", 4, "[B,H,S,D]");
  require_rank(in, k, "k", 4, "[B,H,S,D]");
  TORCH_CHECK(v.sizes() == k.sizes(), "masked_attention: k and v must have the same shape, got ",
              k.sizes(), " and ", v.sizes());
  const int batch = extent(in.op(), "batch", q.size(0));
  const int heads = extent(in.op(), "heads", q.size(1));
  const int seq = extent(in.op(), "sequence", q.size(2));
  const int dim = extent(in.op(), "head dimension", q.size(3));
  const int kv_heads = extent(in.op(), "key heads", k.size(1));
  TORCH_CHECK(k.size(0) == batch && k.size(2) == seq && k.size(3) == dim,
              "masked_attention: q and k must have the same shape but for their heads, got ",
              q.sizes(), " and ", k.sizes());
  check_heads(in, heads, kv_heads, dim);
  check_slopes(in, slopes, heads);
  if (documents) {
    require_aux(in, *documents, "documents", at::kInt);
    TORCH_CHECK(documents->dim() == 2 && documents->size(0) == batch && documents->size(1) == seq,
                "masked_attention: documents must be [batch, sequence], got ", documents->sizes());
  }
  if (prefixes) {
    require_aux(in, *prefixes, "prefixes", at::kInt);
    TORCH_CHECK(prefixes->dim() == 1 && prefixes->size(0) == batch,
                "masked_attention: prefixes must be [batch], got ", prefixes->sizes());
  }
  const float sc = scale_of(in, scale, dim), cap = softcap_of(in, softcap);
  const int win = window_of(in, window);
  const operatorlib_strides_t qs = strides_of(in, q, "q"), ks = strides_of(in, k, "k"),
                              vs = strides_of(in, v, "v");
  at::Tensor out = at::empty_like(q);  // q's order of dimensions, dense
  const operatorlib_strides_t os = strides_of(in, out, "output");
  launch(in, [&](void* s) {
    return in.half()
               ? operatorlib_masked_attention_f16(half_in(q), qs, half_in(k), ks, half_in(v), vs,
                                                  floats(slopes), ints(documents), ints(prefixes),
                                                  half_out(out), os, batch, heads, kv_heads, seq,
                                                  dim, sc, causal, win, cap, s)
               : operatorlib_masked_attention_f32(float_in(q), qs, float_in(k), ks, float_in(v),
                                                  vs, floats(slopes), ints(documents),
                                                  ints(prefixes), float_out(out), os, batch, heads,
                                                  kv_heads, seq, dim, sc, causal, win, cap, s);
  });
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(operatorlib, m) {
  m.def("rope_append(Tensor q, Tensor k, Tensor v, Tensor positions, Tensor frequencies, "
        "Tensor slots, Tensor(a!) key_cache, Tensor(b!) value_cache, *, Tensor? axes=None, "
        "bool interleaved=False, bool return_keys=False) -> (Tensor, Tensor)");
  m.def("paged_attention(Tensor q, Tensor key_cache, Tensor value_cache, Tensor page_table, "
        "Tensor lengths, *, float? scale=None, int window=0, float softcap=0.0, "
        "Tensor? slopes=None) -> Tensor");
  m.def("masked_attention(Tensor q, Tensor k, Tensor v, *, bool causal=False, int window=0, "
        "float softcap=0.0, Tensor? slopes=None, Tensor? documents=None, Tensor? prefixes=None, "
        "float? scale=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(operatorlib, CUDA, m) {
  m.impl("rope_append", &rope_append_op);
  m.impl("paged_attention", &paged_attention_op);
  m.impl("masked_attention", &masked_attention_op);
}
