// rope_append: rotates a step's queries and keys and stores its keys and
// values in a paged cache (operatorlib/lm_c.h).
//
// Pair (a, b) of a head -> (a cos t - b sin t, b cos t + a sin t) with
// t = position * frequency. The product is taken in 64 bits and reduced to a
// fraction of a turn there: in 32 bits position 131072 times frequency 1
// would leave an angle known to 2^-8 radians. cos and sin of the fraction
// are taken in fp32 (an error of 2^-24 of a turn before, 2 ulp after), the
// rotation in fp32, each output rounded to its type once.
//
// Every element is read once and written once or twice: bound by HBM (8192 tokens
// of 32 + 8 heads of 128 in fp16: 37.4 us, 5.8 TB/s; a 1 GiB copy runs at 5.2).
// One workgroup handles a token, or a share of its elements when there are few
// tokens; 16-byte chunks, one rotation item being two chunks half a rotary width
// apart (or one chunk of neighbouring pairs). The cos / sin table of the token is
// computed once per workgroup into LDS while the first chunks are in flight, and
// serves all of its query and key heads. A step of 64 tokens takes 3.1 us, of
// which an empty launch is 1.7.

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "common.hpp"
#include "divide.hpp"
#include "lm_validate.hpp"
#include "operatorlib/lm_c.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTable = 512;  // pairs of the LDS table; wider rotations compute per item

template <typename T, int E>
struct Chunk {
  typedef T type __attribute__((ext_vector_type(E)));
};
template <typename T>
struct Chunk<T, 1> {
  struct type {
    T v;
    __device__ T& operator[](int) { return v; }
    __device__ const T& operator[](int) const { return v; }
  };
};

template <bool kStream, typename C>
__device__ __forceinline__ void store(C* to, const C& x) {
  if constexpr (kStream)
    __builtin_nontemporal_store(x, to);
  else
    *to = x;
}

// Outputs from this size on, past the 32 MiB of the L2s, are stored
// non-temporally: 8192 tokens of 32 + 8 heads of 128 in fp16 (118 MB) 42.3 -> 37.4 us,
// 4001 of 12 + 12 heads of 80 in fp32 (61 MB) 22.9 -> 18.7. Smaller ones stay for the
// attention that reads them next.
constexpr std::size_t kStreamBytes = std::size_t(32) << 20;

template <typename T>
struct RopeArgs {
  const T* q;
  const T* k;
  const T* v;
  std::int64_t q_stride, k_stride, v_stride;
  const std::int32_t* positions;
  const std::int32_t* axes;
  const float* frequencies;
  const std::int32_t* slots;
  T* q_out;
  T* k_out;
  T* key_cache;
  T* value_cache;
  int tokens, position_rows, q_heads, kv_heads, head_dim, rotary_dim, cache_slots, page_size;
  int parts;  // workgroups per token
  opl::Divider of_part, of_rotated, of_tail, of_whole;  // by parts; by a head's items of each kind
};

// cos and sin of pair i's angle at token t.
template <typename T>
__device__ __forceinline__ float2 unit_of(const RopeArgs<T>& a, int t, int i) {
  const int axis = a.axes == nullptr ? 0 : a.axes[i];
  if (axis < 0 || axis >= a.position_rows) return make_float2(1.0f, 0.0f);
  const double angle =
      static_cast<double>(a.positions[static_cast<std::int64_t>(axis) * a.tokens + t]) *
      static_cast<double>(a.frequencies[i]);
  const double turns = angle * 0.15915494309189533577;  // 1 / (2 pi)
  float s, c;
  sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
  return make_float2(c, s);
}

// E: elements per access (a whole 16-byte chunk, or 1 on unaligned tensors).
// kStream: stores that keep nothing in the caches.
template <typename T, int E, bool kInterleaved, bool kStream>
__global__ __launch_bounds__(kThreads) void rope_append_kernel(const RopeArgs<T> a) {
  using C = typename Chunk<T, E>::type;
  // Pair items: half-split, chunks (i, i + R / 2); interleaved, one chunk of
  // E / 2 pairs (E = 1: the two elements of one pair).
  constexpr int kPairs = kInterleaved ? (E == 1 ? 1 : E / 2) : E;  // pairs per item
  constexpr bool kTwo = !kInterleaved || E == 1;                   // two accesses per item
  __shared__ float2 table[kMaxTable];

  const int t = a.of_part.quotient(static_cast<int>(blockIdx.x));
  const int part = static_cast<int>(blockIdx.x) - t * a.parts;
  const int pairs = a.rotary_dim / 2;
  const bool in_table = pairs <= kMaxTable;
  const std::int64_t d = a.head_dim;

  // Items: [pair items of q heads, of k heads][copied chunks past the rotary
  // dims of q and k heads][chunks of v heads].
  const int per_head = pairs / kPairs;
  const int tail = (a.head_dim - a.rotary_dim) / E;
  const int whole = a.head_dim / E;
  const int qk = a.q_heads + a.kv_heads;
  const int rotated = qk * per_head;
  const int copied = rotated + qk * tail;
  const int total = copied + a.kv_heads * whole;

  // An item's head (of q, then k, then v), its first chunk's dim and its second's.
  struct Item {
    int head, lo, hi;
    bool rotate;
  };
  auto item_of = [&](int i) {
    Item m;
    m.rotate = i < rotated;
    if (m.rotate) {
      m.head = a.of_rotated.quotient(i);
      const int first = (i - m.head * per_head) * kPairs;  // pair
      m.lo = kInterleaved ? 2 * first : first;
      m.hi = kInterleaved ? m.lo + 1 : m.lo + pairs;
    } else if (i < copied) {
      m.head = a.of_tail.quotient(i - rotated);
      m.lo = a.rotary_dim + (i - rotated - m.head * tail) * E;
    } else {
      m.head = a.of_whole.quotient(i - copied);
      m.lo = (i - copied - m.head * whole) * E;
      m.head += qk;
    }
    return m;
  };
  // The first kBatch items of each thread are read before the angles are
  // computed, and every further batch before its first is stored. Items of two
  // chunks one at a time, as registers cost wavefronts (8192 tokens, 32 + 8 heads of
  // 128: 42.4 us, 44.1 with two, 44.3 with three); of one chunk three (4001 tokens,
  // 12 + 12 heads of 80 in fp32: 25.1 us with one, 23.8 with two, 22.9).
  constexpr int kBatch = kTwo ? 1 : 3;
  C x[kBatch], y[kBatch];
  auto read = [&](int i0) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = i0 + k * a.parts * kThreads;
      if (i >= total) continue;
      const Item m = item_of(i);
      const T* src = m.head < a.q_heads ? a.q + t * a.q_stride + m.head * d
                     : m.head < qk      ? a.k + t * a.k_stride + (m.head - a.q_heads) * d
                                        : a.v + t * a.v_stride + (m.head - qk) * d;
      x[k] = *reinterpret_cast<const C*>(src + m.lo);
      if constexpr (kTwo)
        if (m.rotate) y[k] = *reinterpret_cast<const C*>(src + m.hi);
    }
  };
  const int first_item = part * kThreads + static_cast<int>(threadIdx.x);
  read(first_item);

  const int slot = a.slots[t];
  if (in_table) {
    for (int i = threadIdx.x; i < pairs; i += kThreads) table[i] = unit_of(a, t, i);
    __syncthreads();
  }
  const bool stored = slot >= 0 && slot < a.cache_slots;
  const int page = stored ? slot / a.page_size : 0;
  const int row = stored ? slot - page * a.page_size : 0;
  const std::int64_t cache_row =
      (static_cast<std::int64_t>(page) * a.kv_heads * a.page_size + row) * d;
  const std::int64_t cache_head = a.page_size * d;

  for (int i0 = first_item; i0 < total; i0 += kBatch * a.parts * kThreads) {
    if (i0 != first_item) read(i0);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = i0 + k * a.parts * kThreads;
      if (i >= total) continue;
      const Item m = item_of(i);
      if (m.rotate) {
        const int first = kInterleaved ? m.lo / 2 : m.lo;
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          const float2 u = in_table ? table[first + e] : unit_of(a, t, first + e);
          if constexpr (kTwo) {
            const float p = static_cast<float>(x[k][e]), q = static_cast<float>(y[k][e]);
            x[k][e] = static_cast<T>(p * u.x - q * u.y);
            y[k][e] = static_cast<T>(q * u.x + p * u.y);
          } else {
            const float p = static_cast<float>(x[k][2 * e]), q = static_cast<float>(x[k][2 * e + 1]);
            x[k][2 * e] = static_cast<T>(p * u.x - q * u.y);
            x[k][2 * e + 1] = static_cast<T>(q * u.x + p * u.y);
          }
        }
      }
      auto write = [&](T* to) {
        store<kStream>(reinterpret_cast<C*>(to + m.lo), x[k]);
        if constexpr (kTwo)
          if (m.rotate) store<kStream>(reinterpret_cast<C*>(to + m.hi), y[k]);
      };
      if (m.head < a.q_heads) {
        write(a.q_out + (static_cast<std::int64_t>(t) * a.q_heads + m.head) * d);
      } else if (m.head < qk) {
        const int h = m.head - a.q_heads;
        if (a.k_out != nullptr) write(a.k_out + (static_cast<std::int64_t>(t) * a.kv_heads + h) * d);
        if (stored) write(a.key_cache + cache_row + h * cache_head);
      } else if (stored) {
        write(a.value_cache + cache_row + (m.head - qk) * cache_head);
      }
    }
  }
}

template <typename T, int E>
hipError_t launch(RopeArgs<T> a, bool interleaved, hipStream_t stream) {
  const int pairs = a.rotary_dim / 2;
  const long long per_head =
      interleaved && E > 1 ? pairs / (E / 2) : pairs / E;
  const long long items =
      (a.q_heads + a.kv_heads) * (per_head + (a.head_dim - a.rotary_dim) / E) +
      static_cast<long long>(a.kv_heads) * (a.head_dim / E);
  // Few tokens: a workgroup per 256 items, so that a step of few sequences
  // spreads over the CUs; many tokens: one workgroup each.
  long long parts = (items + kThreads - 1) / kThreads;
  const long long spread = (1024 + a.tokens - 1) / a.tokens;
  if (parts > spread) parts = spread;
  a.parts = static_cast<int>(parts);
  const auto divider = [](long long n) { return opl::Divider::by(n > 0 ? static_cast<int>(n) : 1); };
  a.of_part = divider(parts);
  a.of_rotated = divider(per_head);
  a.of_tail = divider((a.head_dim - a.rotary_dim) / E);
  a.of_whole = divider(a.head_dim / E);
  const dim3 grid(static_cast<unsigned>(parts * a.tokens));
  const std::size_t row = static_cast<std::size_t>(a.q_heads) + (a.k_out != nullptr ? 3 : 2) * a.kv_heads;
  if (E > 1 && row * a.head_dim * a.tokens * sizeof(T) >= kStreamBytes) {
    if constexpr (E > 1) {
      if (interleaved)
        rope_append_kernel<T, E, true, true><<<grid, dim3(kThreads), 0, stream>>>(a);
      else
        rope_append_kernel<T, E, false, true><<<grid, dim3(kThreads), 0, stream>>>(a);
    }
  } else if (interleaved) {
    rope_append_kernel<T, E, true, false><<<grid, dim3(kThreads), 0, stream>>>(a);
  } else {
    rope_append_kernel<T, E, false, false><<<grid, dim3(kThreads), 0, stream>>>(a);
  }
  return hipGetLastError();
}

template <typename T>
int rope_entry(RopeArgs<T> a, int interleaved, int pages, void* stream_handle) {
  const opl::RopeShape shape = {a.q_stride, a.k_stride,  a.v_stride,   a.position_rows, a.tokens,
                                a.q_heads,  a.kv_heads,  a.head_dim,   a.rotary_dim,    pages,
                                a.page_size};
  if (a.q == nullptr || a.k == nullptr || a.v == nullptr || a.slots == nullptr ||
      a.q_out == nullptr || a.key_cache == nullptr || a.value_cache == nullptr ||
      !opl::rope_shape_ok(shape))
    return hipErrorInvalidValue;
  // (a cache's bytes fit 63 bits: slots and a token's elements fit 31 each)
  const std::uint64_t cache_bytes = static_cast<std::uint64_t>(pages) * a.page_size * a.kv_heads * a.head_dim * sizeof(T);
  const auto key_at = reinterpret_cast<std::uintptr_t>(a.key_cache), value_at = reinterpret_cast<std::uintptr_t>(a.value_cache);
  if ((key_at < value_at ? value_at - key_at : key_at - value_at) < cache_bytes) return hipErrorInvalidValue;
  if (a.rotary_dim > 0 && (a.positions == nullptr || a.frequencies == nullptr))
    return hipErrorInvalidValue;
  a.cache_slots = pages * a.page_size;
  constexpr int E = 16 / sizeof(T);
  const int unit = interleaved ? a.rotary_dim : a.rotary_dim / 2;
  const bool chunks = a.head_dim % E == 0 && unit % E == 0 &&
                      opl::aligned_rows(a.q, sizeof(T), a.q_stride) &&
                      opl::aligned_rows(a.k, sizeof(T), a.k_stride) &&
                      opl::aligned_rows(a.v, sizeof(T), a.v_stride) &&
                      opl::aligned16(a.q_out) && opl::aligned16(a.k_out) &&
                      opl::aligned16(a.key_cache) && opl::aligned16(a.value_cache);
  const hipStream_t stream = static_cast<hipStream_t>(stream_handle);
  return chunks ? launch<T, E>(a, interleaved != 0, stream)
                : launch<T, 1>(a, interleaved != 0, stream);
}

}  // namespace

extern "C" int operatorlib_lm_abi_version(void) { return OPERATORLIB_LM_ABI_VERSION; }

extern "C" int operatorlib_rope_append_f16(
    const operatorlib_half_t* q, int64_t q_token_stride, const operatorlib_half_t* k,
    int64_t k_token_stride, const operatorlib_half_t* v, int64_t v_token_stride,
    const int32_t* positions, int position_rows, const int32_t* axes, const float* frequencies,
    const int32_t* slots, operatorlib_half_t* q_out, operatorlib_half_t* k_out,
    operatorlib_half_t* key_cache, operatorlib_half_t* value_cache, int tokens, int q_heads,
    int kv_heads, int head_dim, int rotary_dim, int interleaved, int pages, int page_size,
    void* stream) {
  const auto in = [](const operatorlib_half_t* p) { return reinterpret_cast<const _Float16*>(p); };
  const auto out = [](operatorlib_half_t* p) { return reinterpret_cast<_Float16*>(p); };
  return rope_entry<_Float16>(
      {in(q), in(k), in(v), q_token_stride, k_token_stride, v_token_stride, positions, axes,
       frequencies, slots, out(q_out), out(k_out), out(key_cache), out(value_cache), tokens,
       position_rows, q_heads, kv_heads, head_dim, rotary_dim, 0, page_size, 1},
      interleaved, pages, stream);
}

extern "C" int operatorlib_rope_append_f32(
    const float* q, int64_t q_token_stride, const float* k, int64_t k_token_stride, const float* v,
    int64_t v_token_stride, const int32_t* positions, int position_rows, const int32_t* axes,
    const float* frequencies, const int32_t* slots, float* q_out, float* k_out, float* key_cache,
    float* value_cache, int tokens, int q_heads, int kv_heads, int head_dim, int rotary_dim,
    int interleaved, int pages, int page_size, void* stream) {
  return rope_entry<float>(
      {q, k, v, q_token_stride, k_token_stride, v_token_stride, positions, axes, frequencies,
       slots, q_out, k_out, key_cache, value_cache, tokens, position_rows, q_heads, kv_heads,
       head_dim, rotary_dim, 0, page_size, 1},
      interleaved, pages, stream);
}
