#pragma once
// operatorlib C++ API, language-model operators: inline forwarders to the C ABI
// of operatorlib/lm_c.h (liboperatorlib_lm.so), which documents them, with
// hipError_t / hipStream_t / __half, as operatorlib/operators.h is for the
// other operators. What is optional comes last and has a default.

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

#include "operatorlib/lm_c.h"

namespace operatorlib {

// A strided operand: its first element and the distances of lm_c.h.
template <typename T>
struct TokenRows {  // [tokens, heads, head_dim], tokens `stride` elements apart
  T* data;
  std::int64_t stride;
};

struct RopeAppendShape {
  int tokens, q_heads, kv_heads, head_dim, rotary_dim, pages, page_size;
};

namespace lm_detail {
inline const operatorlib_half_t* bits(const __half* p) {
  return reinterpret_cast<const operatorlib_half_t*>(p);
}
inline operatorlib_half_t* bits(__half* p) { return reinterpret_cast<operatorlib_half_t*>(p); }
}  // namespace lm_detail

inline hipError_t rope_append_f16(TokenRows<const __half> q, TokenRows<const __half> k,
                                  TokenRows<const __half> v, const std::int32_t* positions,
                                  const float* frequencies, const std::int32_t* slots,
                                  __half* q_out, __half* key_cache, __half* value_cache,
                                  const RopeAppendShape& s, __half* k_out = nullptr,
                                  const std::int32_t* axes = nullptr, int position_rows = 1,
                                  bool interleaved = false, hipStream_t stream = nullptr) {
  using lm_detail::bits;
  return static_cast<hipError_t>(operatorlib_rope_append_f16(
      bits(q.data), q.stride, bits(k.data), k.stride, bits(v.data), v.stride, positions,
      position_rows, axes, frequencies, slots, bits(q_out), bits(k_out), bits(key_cache),
      bits(value_cache), s.tokens, s.q_heads, s.kv_heads, s.head_dim, s.rotary_dim,
      interleaved ? 1 : 0, s.pages, s.page_size, static_cast<void*>(stream)));
}

inline hipError_t rope_append_f32(TokenRows<const float> q, TokenRows<const float> k,
                                  TokenRows<const float> v, const std::int32_t* positions,
                                  const float* frequencies, const std::int32_t* slots,
                                  float* q_out, float* key_cache, float* value_cache,
                                  const RopeAppendShape& s, float* k_out = nullptr,
                                  const std::int32_t* axes = nullptr, int position_rows = 1,
                                  bool interleaved = false, hipStream_t stream = nullptr) {
  return static_cast<hipError_t>(operatorlib_rope_append_f32(
      q.data, q.stride, k.data, k.stride, v.data, v.stride, positions, position_rows, axes,
      frequencies, slots, q_out, k_out, key_cache, value_cache, s.tokens, s.q_heads, s.kv_heads,
      s.head_dim, s.rotary_dim, interleaved ? 1 : 0, s.pages, s.page_size,
      static_cast<void*>(stream)));
}

struct PagedShape {
  int batch, q_heads, kv_heads, head_dim, pages, page_size, max_pages;
};

// q [batch, q_heads, head_dim] and page_table [batch, max_pages] dense here;
// the C ABI takes their strides.
inline hipError_t paged_attention_f16(const __half* q, const __half* key_cache,
                                      const __half* value_cache, const std::int32_t* page_table,
                                      const std::int32_t* lengths, __half* output,
                                      const PagedShape& s, float scale, int window = 0,
                                      float softcap = 0.0f, const float* slopes = nullptr,
                                      hipStream_t stream = nullptr) {
  using lm_detail::bits;
  return static_cast<hipError_t>(operatorlib_paged_attention_f16(
      bits(q), static_cast<std::int64_t>(s.q_heads) * s.head_dim, bits(key_cache),
      bits(value_cache), page_table, s.max_pages, lengths, slopes, bits(output), s.batch,
      s.q_heads, s.kv_heads, s.head_dim, s.pages, s.page_size, s.max_pages, scale, window, softcap,
      static_cast<void*>(stream)));
}

inline hipError_t paged_attention_f32(const float* q, const float* key_cache,
                                      const float* value_cache, const std::int32_t* page_table,
                                      const std::int32_t* lengths, float* output,
                                      const PagedShape& s, float scale, int window = 0,
                                      float softcap = 0.0f, const float* slopes = nullptr,
                                      hipStream_t stream = nullptr) {
  return static_cast<hipError_t>(operatorlib_paged_attention_f32(
      q, static_cast<std::int64_t>(s.q_heads) * s.head_dim, key_cache, value_cache, page_table,
      s.max_pages, lengths, slopes, output, s.batch, s.q_heads, s.kv_heads, s.head_dim, s.pages,
      s.page_size, s.max_pages, scale, window, softcap, static_cast<void*>(stream)));
}

struct MaskedShape {
  int batch, q_heads, kv_heads, sequence, head_dim;
};

// The rules of masked_attention; the defaults show every key to every query.
struct MaskRules {
  bool causal = false;
  int window = 0;
  float softcap = 0.0f;
  const float* slopes = nullptr;
  const std::int32_t* documents = nullptr;
  const std::int32_t* prefixes = nullptr;
};

// Contiguous [B, H, S, D] tensors here; the C ABI takes their strides.
inline hipError_t masked_attention_f16(const __half* q, const __half* k, const __half* v,
                                       __half* output, const MaskedShape& s, float scale,
                                       const MaskRules& r = {}, hipStream_t stream = nullptr) {
  using lm_detail::bits;
  const std::int64_t head = static_cast<std::int64_t>(s.sequence) * s.head_dim;
  const operatorlib_strides_t qs = {s.q_heads * head, head, s.head_dim};
  const operatorlib_strides_t ks = {s.kv_heads * head, head, s.head_dim};
  return static_cast<hipError_t>(operatorlib_masked_attention_f16(
      bits(q), qs, bits(k), ks, bits(v), ks, r.slopes, r.documents, r.prefixes, bits(output), qs,
      s.batch, s.q_heads, s.kv_heads, s.sequence, s.head_dim, scale, r.causal ? 1 : 0, r.window,
      r.softcap, static_cast<void*>(stream)));
}

inline hipError_t masked_attention_f32(const float* q, const float* k, const float* v,
                                       float* output, const MaskedShape& s, float scale,
                                       const MaskRules& r = {}, hipStream_t stream = nullptr) {
  const std::int64_t head = static_cast<std::int64_t>(s.sequence) * s.head_dim;
  const operatorlib_strides_t qs = {s.q_heads * head, head, s.head_dim};
  const operatorlib_strides_t ks = {s.kv_heads * head, head, s.head_dim};
  return static_cast<hipError_t>(operatorlib_masked_attention_f32(
      q, qs, k, ks, v, ks, r.slopes, r.documents, r.prefixes, output, qs, s.batch, s.q_heads,
      s.kv_heads, s.sequence, s.head_dim, scale, r.causal ? 1 : 0, r.window, r.softcap,
      static_cast<void*>(stream)));
}

}  // namespace operatorlib
