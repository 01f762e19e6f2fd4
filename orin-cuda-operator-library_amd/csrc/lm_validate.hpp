#pragma once
// Argument predicates of the language-model entry points
// (operatorlib/lm_c.h). Pure C++ with no HIP calls, as validate.hpp.

#include <cmath>
#include <cstddef>
#include <cstdint>
#include <limits>

#include "validate.hpp"

namespace opl {

constexpr std::int64_t kInt32Max = std::numeric_limits<std::int32_t>::max();

// A launch holds less than 2^32 threads: workgroups of 256 that always fit.
constexpr std::int64_t kMostWorkgroups = (1 << 24) - 8;

// Sizes, strides and flags of a rope_append call.
struct RopeShape {
  std::int64_t q_stride, k_stride, v_stride;
  int position_rows, tokens, q_heads, kv_heads, head_dim, rotary_dim, pages, page_size;
};

inline bool rope_shape_ok(const RopeShape& s) {
  if (s.tokens <= 0 || s.tokens > kMostWorkgroups || s.q_heads <= 0 || s.kv_heads <= 0 || s.head_dim <= 0 || s.pages <= 0 ||
      s.page_size <= 0 || s.rotary_dim < 0 || s.rotary_dim % 2 != 0 || s.rotary_dim > s.head_dim)
    return false;
  if (s.rotary_dim > 0 && s.position_rows <= 0) return false;
  if (static_cast<std::int64_t>(s.pages) * s.page_size > kInt32Max) return false;
  const std::int64_t q_row = static_cast<std::int64_t>(s.q_heads) * s.head_dim;
  const std::int64_t kv_row = static_cast<std::int64_t>(s.kv_heads) * s.head_dim;
  // A token's elements are counted in 32 bits by the kernel, in steps of up to
  // 3 x 1024 workgroups of 256.
  if (q_row > kInt32Max || kv_row > kInt32Max || q_row + 2 * kv_row > kInt32Max - (1 << 20))
    return false;
  return s.q_stride >= q_row && s.k_stride >= kv_row && s.v_stride >= kv_row;
}

// The rules that turn a dot product into a score. The kernels multiply by
// scale, by scale / softcap and by softcap, each times up to 2 log2 e, and by their
// inverses: none may leave the range of fp32.
inline bool within_rules(float x) { return x >= 0x1p-100f && x <= 0x1p100f; }
inline bool score_rules_ok(float scale, int window, float softcap) {
  return within_rules(scale) && window >= 0 &&
         (softcap == 0.0f || (within_rules(softcap) && within_rules(scale / softcap)));
}

inline bool aligned_rows(const void* p, std::size_t element_bytes, std::int64_t stride) {
  return (reinterpret_cast<std::uintptr_t>(p) & 15u) == 0 &&
         stride % static_cast<std::int64_t>(16 / element_bytes) == 0;
}

// Keys of a unit of paged attention work: what the four wavefronts of a
// workgroup read together in one step (paged_attention.hip).
inline constexpr int paged_unit_keys(std::size_t element_bytes) {
  return element_bytes == 2 ? 128 : 64;
}
// Query heads that share a key head and are computed by one workgroup.
constexpr int kPagedHeads = 32;

struct PagedShape {
  int batch, q_heads, kv_heads, head_dim, page_size, max_pages;
};

inline bool paged_shape_ok(const PagedShape& s, std::size_t element_bytes) {
  if (s.batch <= 0 || s.q_heads <= 0 || s.kv_heads <= 0 || s.head_dim <= 0 ||
      s.head_dim > kMaxHeadDim || s.page_size <= 0 || s.max_pages <= 0)
    return false;
  if (s.q_heads % s.kv_heads != 0 ||
      s.head_dim % static_cast<int>(16 / element_bytes) != 0)
    return false;
  const std::int64_t tokens = static_cast<std::int64_t>(s.max_pages) * s.page_size;
  // (A step past the last token still fits 32 bits.)
  if (tokens > kInt32Max - 1024 || static_cast<std::int64_t>(s.batch) * s.q_heads > kInt32Max)
    return false;
  // batch * q_heads fits 31 bits and tokens 31 bits: no overflow in 64.
  const int tiles = (s.q_heads / s.kv_heads + kPagedHeads - 1) / kPagedHeads;
  return static_cast<std::int64_t>(s.batch) * s.kv_heads * tiles * ((tokens + 63) / 64) <=
         kInt32Max;
}

inline bool paged_cache_ok(int pages, int kv_heads, int page_size) {
  // (64-bit: two factors of 31 bits, then a third once that is in range)
  if (pages <= 0) return false;
  const std::uint64_t rows = static_cast<std::uint64_t>(pages) * page_size;
  const std::uint64_t most = std::numeric_limits<std::uint32_t>::max();
  return rows <= most && rows * static_cast<std::uint64_t>(kv_heads) <= most;
}

struct MaskedShape {
  int batch, q_heads, kv_heads, sequence, head_dim;
};

constexpr int kMaxMaskedSequence = 1 << 20;

inline bool masked_shape_ok(const MaskedShape& s, std::size_t element_bytes) {
  if (s.batch <= 0 || s.q_heads <= 0 || s.kv_heads <= 0 || s.sequence <= 0 ||
      s.sequence > kMaxMaskedSequence || s.head_dim <= 0 || s.head_dim > kMaxHeadDim)
    return false;
  if (s.q_heads % s.kv_heads != 0 ||
      s.head_dim % static_cast<int>(16 / element_bytes) != 0)
    return false;
  const std::int64_t heads = static_cast<std::int64_t>(s.batch) * s.q_heads;
  return heads <= kMostWorkgroups && heads * ((s.sequence + 31) / 32) <= kMostWorkgroups;
}

struct MaskedStrides {
  std::int64_t batch, head, token;
};

// Strides of one operand. Sizes are checked before.
inline bool masked_strides_ok(const void* p, const MaskedStrides& t, const MaskedShape& s,
                              std::size_t element_bytes) {
  if (t.batch < 0 || t.head < 0 || t.token < s.head_dim) return false;
  if (!aligned_rows(p, element_bytes, t.batch) || !aligned_rows(p, element_bytes, t.head) ||
      !aligned_rows(p, element_bytes, t.token))
    return false;
  // A head, and a tile of 64 rows that ends past it, is addressed with 31-bit
  // byte offsets from its first row.
  const std::int64_t limit = (std::int64_t(1) << 31) / static_cast<std::int64_t>(element_bytes);
  return t.token < limit / (s.sequence > 64 ? s.sequence : 64);
}

}  // namespace opl
