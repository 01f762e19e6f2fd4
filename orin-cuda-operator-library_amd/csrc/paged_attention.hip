// paged_attention: one new token per sequence attends to its paged cache
// (operatorlib/lm_c.h).
//
// Per sequence and key head, the query heads that share it are the columns of
// a 16-column matrix-core operand:
//   S^T = K Q^T,  m' = max(m, x), l' = l 2^(m - m') + sum 2^(x - m'),
//   O^T' = O^T 2^(m - m') + V^T P^T   (x: score in log2 units)
// Keys and values are read once, straight from the cache into the registers
// that the matrix instructions take, and nothing passes through LDS until the
// wavefronts of a workgroup join their results:
//   * lane (col, g) = (l % 16, l / 16) of a wavefront supplies row col and the
//     g-th 16-byte chunk of a step to v_mfma_f32_16x16x32_f16 (16x16x4_f32: four
//     instructions per chunk): a K row's chunk is one load;
//   * the S^T block leaves lane (col, g) with head col and keys 4 g + r: the
//     layout of the P^T operand of V^T P^T if the lane's k slots are those keys.
//     So the lane loads chunk col of the V rows 4 g + r (whole rows per
//     instruction), and the t-th elements of its rows, packed by v_perm_b32,
//     are the V^T operand whose row m is dim (chunk width) m + t;
//   * O^T has head col in the lane, like the running max and sum, so a rescale
//     needs no exchange between lanes.
// The matrix cores run far below their rate (at most 16 columns): the kernel
// is bound by reading the cache. A wavefront has one set of registers for a tile
// (K and V, 16 KiB): the next tile's K is loaded as soon as S^T is computed, its V
// as soon as O^T is, and its page ids a tile earlier, so that loads are in
// flight all the time.
//
// Work split. The host does not know the lengths. The unit of work is four
// tiles (one per wavefront of a workgroup) of one row (sequence, key head).
//   * Few units (the page table's whole width in kDirectUnits): a workgroup per
//     unit, and the pieces of a row are the workgroups of its units.
//   * Else the units that the lengths give form one line, and workgroup w of G
//     takes an equal, contiguous piece of it, whatever mix of long and short
//     sequences it holds; it finds its piece by a scan of the lengths (a few
//     per thread). A row within one piece is written at once; a piece cuts at
//     most its first and its last row: two slots of scratch per workgroup.
// The pieces of a row leave unnormalised O with their max and sum, and
// paged_join_kernel adds them in order (deterministic).
//
// Measured on MI355X, fp16, head_dim 128:
//   * 64 sequences of 1 to 8192 tokens, 32 + 8 heads (1.18 GB of cache): 194 us,
//     6.1 TB/s (a 1 GiB copy moves 5.2); 512 workgroups are the two that fit a CU
//     with 2 x 16 KiB in flight per SIMD (three a CU spilled registers).
//   * 2 of 131072 tokens, 16 + 2 heads (263 MB): 57.6 us, of which the join is 6.
//   * 1 of 1000 tokens, 32 + 8 heads: 10.1 us, the chain length -> page -> K -> V ->
//     partial, twice a launch (1.7), and the join's two reads. The last workgroup of
//     a row joining instead of a launch took 11.6 us (15.3 with agent-scope
//     fences); looking pages up before the lengths arrive gained nothing.

#include <hip/hip_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "common.hpp"
#include "divide.hpp"
#include "lm_validate.hpp"
#include "operatorlib/lm_c.h"
#include "scores.hpp"
#include "scratch.hpp"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = 4;
// Workgroups of a launch that shares the units out, and the most units that get
// a workgroup each: what one round holds. (32 + 8 heads, one sequence of 4000 tokens:
// direct 10.4 us, shared out 14.0; of 8100: 12.9, 16.5; 4 of 2000: 12.8, 17.9. In two
// rounds, one of 16000 tokens: direct 23.3, shared out 23.0.)
constexpr int kWorkgroups = 512;
constexpr int kDirectUnits = 512;
// Caches from this size on, three quarters of the 256 MiB Infinity Cache, are read
// with non-temporal loads: they cannot stay there from one step to the next
// beside anything else. Batch of 64 (1.18 GB) 221 -> 195 us (6.0 TB/s), one
// sequence of 131072 tokens (537 MB) 107 -> 97; 263 MB 62.7 -> 57.4 after other
// work, 52.4 -> 57.1 where the step before had left them there; 137 MB 33.3 -> 36.7.
constexpr std::uint64_t kStreamBytes = std::uint64_t(192) << 20;
// Shared-out rows below which a head's pieces, 16 and more, are added by all
// wavefronts of a workgroup (8 rows: 23.0 us, 29.5 with one wavefront per head; 4
// rows, 54.1 -> 33.3), not by one (32 rows: 23.5 us, 21.9 with one; 64 rows: 35.3, 29.7).
constexpr unsigned kFewRows = 32;
// The fp16 form's probabilities are 2^(x - m + kBoost), m the running max less
// at most kLazy: keys far below the max keep 10 more binary orders before they
// become fp16 subnormals, and 2^(kBoost + kLazy) is far below fp16's largest.
constexpr float kBoost = 10.0f;
constexpr float kLazy = 4.0f;

template <typename T, int DP>
struct Shape {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int E = 16 / static_cast<int>(sizeof(T));
  static constexpr int kKeys = kHalf ? 32 : 16;    // keys of a wavefront's tile
  static constexpr int kSubs = kKeys / 16;
  static constexpr int kSteps = DP / (4 * E);      // chunks of a K row per lane
  static constexpr int kVW = DP / 16 < E ? DP / 16 : E;  // elements of a V chunk
  static constexpr int kVC = DP / 16 / kVW;        // V chunks of a row per lane
  static constexpr int kBlocks = DP / 16;          // 16-dim blocks of O^T
  static constexpr int kVRows = kHalf ? 8 : 4;     // V rows per lane
  typedef T KFrag __attribute__((ext_vector_type(E)));
  typedef T VFrag __attribute__((ext_vector_type(kVW)));
  struct Tile {
    KFrag k[kSubs][kSteps];
    VFrag v[kVRows][kVC];
  };
};

template <typename T>
struct PagedArgs {
  const T* q;
  const T* key_cache;
  const T* value_cache;
  const std::int32_t* page_table;
  const std::int32_t* lengths;
  const float* slopes;
  T* out;
  float* part;          // [slots][heads of a row][DP + 4]: O, max, sum; two slots per
                        // workgroup, or (direct) one
  std::int32_t* cut;    // [workgroups][2]: of the row that starts in the workgroup and
                        // ends in a later one, the row and that one; else -1. Direct: NULL
  int direct;           // units of a row that have a workgroup each; 0: shared out
  opl::Divider page_of; // key / page_size
  std::int64_t q_stride, table_stride;
  int batch, q_heads, kv_heads, group, tiles_of_heads, head_dim, pages, page_size, max_pages;
  int window;
  opl::ScoreRules rules;
};

// Visible keys [lo, n) of sequence b.
template <typename T>
__device__ __forceinline__ int2 key_range(const PagedArgs<T>& a, int b) {
  const int n = min(max(a.lengths[b], 0), a.max_pages * a.page_size);
  const int lo = a.window > 0 && n > a.window ? n - a.window : 0;
  return make_int2(lo, n);
}

// Units of a row of sequence b: keys from the tile border below lo.
template <int kUnitKeys>
__device__ __forceinline__ int units_of(int2 r) {
  const int from = r.x & ~15;
  return max(1, (r.y - from + kUnitKeys - 1) / kUnitKeys);
}

template <bool kStream, typename V>
__device__ __forceinline__ V fetch(const V* p) {
  if constexpr (kStream) return __builtin_nontemporal_load(p);
  return *p;
}

// MT: 16-head operands per workgroup (group up to 16 MT). kPaged16: pages hold
// whole 16-key blocks, so that a block's rows follow each other.
// kStream: the cache is read past the caches' reach, with non-temporal loads.
// kWideCap: fp16, capped in the precise form (two sequences of 131072 tokens 58.6 us
// with it, 56.7 without).
template <typename T, int DP, int MT, bool kPaged16, bool kStream, bool kWideCap>
__global__ __launch_bounds__(kThreads) void paged_attention_kernel(const PagedArgs<T> a) {
  using S = Shape<T, DP>;
  constexpr bool kHalf = S::kHalf;
  constexpr int kHeads = 16 * MT;
  constexpr int kUnitKeys = kWaves * S::kKeys;
  constexpr int kPitch = DP + 4;  // floats of a head's row in LDS: rows 16 bytes apart in the banks
  __shared__ __attribute__((aligned(16))) float joined[kWaves][kHeads][kPitch];
  __shared__ int scan[kWaves];
  __shared__ int found[2];

  const int lane = threadIdx.x % opl::kWaveSize;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / opl::kWaveSize);
  const int col = lane % 16;
  const int g = lane / 16;
  const int rows_of = a.kv_heads * a.tiles_of_heads;  // rows of a sequence

  // ---- this workgroup's piece of the units: [unit, end), of which `at` is the
  // first of sequence b
  int unit, end, b, at, total = 0;
  long long G = 0;
  if (a.direct > 0) {
    // In this mode `at` is the first unit of the row's sequence as if every row
    // had a.direct units.
    const int row = blockIdx.x / a.direct;
    b = row / rows_of;
    at = b * rows_of * a.direct;
    unit = blockIdx.x;
    end = unit + 1;
  } else {
    const int chunk = (a.batch + kThreads - 1) / kThreads;
    const int b_first = min(a.batch, static_cast<int>(threadIdx.x) * chunk);
    const int b_last = min(a.batch, b_first + chunk);
    int mine = 0;
    for (int i = b_first; i < b_last; ++i) mine += units_of<kUnitKeys>(key_range(a, i)) * rows_of;
    int upto = mine;  // inclusive scan over the wavefront, then over the four
#pragma unroll
    for (int step = 1; step < opl::kWaveSize; step *= 2) {
      const int below = __shfl_up(upto, step);
      if (lane >= step) upto += below;
    }
    if (lane == opl::kWaveSize - 1) scan[wave] = upto;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) upto += scan[w];
      total += scan[w];
    }
    // (No more pieces than units: each of a cut row's workgroups has a part of it.)
    G = min(static_cast<int>(gridDim.x), total);
    if (blockIdx.x >= G) {
      if (a.cut != nullptr && threadIdx.x == 0) a.cut[2 * blockIdx.x] = -1;
      return;
    }
    const int begin = static_cast<int>(static_cast<long long>(blockIdx.x) * total / G);
    end = static_cast<int>((static_cast<long long>(blockIdx.x) + 1) * total / G);
    if (begin >= upto - mine && begin < upto) {
      int first = upto - mine, i = b_first;
      for (;; ++i) {
        const int u = units_of<kUnitKeys>(key_range(a, i)) * rows_of;
        if (begin < first + u) break;
        first += u;
      }
      found[0] = i;
      found[1] = first;
    }
    __syncthreads();
    unit = begin;
    b = __builtin_amdgcn_readfirstlane(found[0]);
    at = __builtin_amdgcn_readfirstlane(found[1]);
    total = __builtin_amdgcn_readfirstlane(total);
  }
  const int begin = unit;
  const int dm = a.head_dim;

  // Offsets (elements) of the lane's chunks in a K and a V row; dims from dm
  // on read dim 0 instead: Q is zero there, and such O dims are not stored.
  int k_dim[S::kSteps], v_dim[S::kVC];
#pragma unroll
  for (int c = 0; c < S::kSteps; ++c) {
    const int d = (4 * c + g) * S::E;
    k_dim[c] = d < dm ? d : 0;
  }
#pragma unroll
  for (int u = 0; u < S::kVC; ++u) {
    const int d = (16 * u + col) * S::kVW;
    v_dim[u] = d < dm ? d : 0;
  }

  while (unit < end) {
    // ---- the row (sequence b, key head, tile of heads) that `unit` lies in
    int2 range = key_range(a, b);
    int units = a.direct > 0 ? a.direct : units_of<kUnitKeys>(range);
    while (unit >= at + units * rows_of) {  // (never in the direct mode)
      at += units * rows_of;
      ++b;
      range = key_range(a, b);
      units = units_of<kUnitKeys>(range);
    }
    const int row_in = (unit - at) / units;
    const int row0 = at + row_in * units;  // first unit of the row
    const int kv_head = row_in / a.tiles_of_heads;
    const int head_tile = row_in % a.tiles_of_heads;
    const int heads = min(kHeads, a.group - head_tile * kHeads);
    const int head0 = kv_head * a.group + head_tile * kHeads;
    const int stop = min(end, row0 + units);
    const int lo = range.x, n = range.y;
    const int base_key = (lo & ~15) + (unit - row0) * kUnitKeys;
    const int last_key = min(n, (lo & ~15) + (stop - row0) * kUnitKeys);

    // ---- Q^T operand
    typename S::KFrag qf[MT][S::kSteps];
    float slope[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int hh = 16 * mt + col;
      const T* qrow = a.q + static_cast<std::int64_t>(b) * a.q_stride +
                      static_cast<std::int64_t>(head0 + (hh < heads ? hh : 0)) * dm;
#pragma unroll
      for (int c = 0; c < S::kSteps; ++c) {
        const int d = (4 * c + g) * S::E;
        qf[mt][c] = *reinterpret_cast<const typename S::KFrag*>(qrow + k_dim[c]);
        if (d >= dm || hh >= heads) qf[mt][c] = typename S::KFrag{};
      }
      slope[mt] = a.slopes != nullptr ? a.slopes[head0 + (hh < heads ? hh : 0)] * opl::kLog2e : 0.0f;
    }

    floatx4 o[MT][S::kBlocks];
    floatx4 sums[MT];
    float row_max[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int i = 0; i < S::kBlocks; ++i) o[mt][i] = floatx4{0, 0, 0, 0};
      sums[mt] = floatx4{0, 0, 0, 0};
      row_max[mt] = -FLT_MAX;
    }

    const std::int32_t* table = a.page_table + static_cast<std::int64_t>(b) * a.table_stride;
    // Page ids of a tile's blocks (kPaged16) or of the lane's K rows; -1 behind
    // the last token.
    struct Pages {
      int id[S::kSubs];
    };
    auto look_up = [&](int key0) {
      Pages p;
#pragma unroll
      for (int s = 0; s < S::kSubs; ++s) {
        const int key = key0 + 16 * s + (kPaged16 ? 0 : col);
        p.id[s] = -1;
        if (key < n) p.id[s] = table[a.page_of.quotient(key)];
      }
      return p;
    };
    // Cache rows of the lane's K and V rows in the tile, and which of the lane's
    // keys are visible (bit 4 s + r: key 16 s + 4 g + r). Hidden keys on no page
    // read the cache's first rows.
    struct Rows {
      std::int64_t sub[S::kSubs];  // kPaged16: first row of each block; else the lane's K rows
      std::int64_t v[kPaged16 ? 1 : S::kVRows];
      unsigned seen;
    };
    auto rows_of_tile = [&](int key0, const Pages& pages) {
      Rows r;
      r.seen = 0;
#pragma unroll
      for (int s = 0; s < S::kSubs; ++s) {
        const int key = key0 + 16 * s + (kPaged16 ? 0 : col);
        const int page = pages.id[s] >= 0 && pages.id[s] < a.pages ? pages.id[s] : -1;
        r.sub[s] = page >= 0 ? (static_cast<std::int64_t>(page) * a.kv_heads + kv_head) * a.page_size +
                                   (key - a.page_of.quotient(key) * a.page_size)
                             : 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int from = 4 * g + e;  // the lane that looked up key 16 s + 4 g + e
          const int mk = key0 + 16 * s + from;
          if constexpr (!kPaged16) r.v[4 * s + e] = __shfl(r.sub[s], from);
          const int its_page = kPaged16 ? page : __shfl(page, from);
          if ((its_page >= 0) & (mk >= lo) & (mk < n)) r.seen |= 1u << (4 * s + e);
        }
      }
      return r;
    };
    auto load_k = [&](typename S::Tile& t, const Rows& r) {
#pragma unroll
      for (int s = 0; s < S::kSubs; ++s) {
        const T* base = a.key_cache + r.sub[s] * dm + (kPaged16 ? col * dm : 0);
#pragma unroll
        for (int c = 0; c < S::kSteps; ++c)
          t.k[s][c] = fetch<kStream>(reinterpret_cast<const typename S::KFrag*>(base + k_dim[c]));
      }
    };
    auto load_v = [&](typename S::Tile& t, const Rows& r) {
#pragma unroll
      for (int j = 0; j < S::kVRows; ++j) {
        const T* base = kPaged16 ? a.value_cache + r.sub[j / 4] * dm + (4 * g + j % 4) * dm
                                 : a.value_cache + r.v[kPaged16 ? 0 : j] * dm;
#pragma unroll
        for (int u = 0; u < S::kVC; ++u)
          t.v[j][u] = fetch<kStream>(reinterpret_cast<const typename S::VFrag*>(base + v_dim[u]));
      }
    };
    floatx4 x[MT][S::kSubs];
    auto scores = [&](const typename S::Tile& t) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int s = 0; s < S::kSubs; ++s) x[mt][s] = floatx4{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < S::kSteps; ++c)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int s = 0; s < S::kSubs; ++s) {
            if constexpr (kHalf) {
              x[mt][s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(t.k[s][c], qf[mt][c], x[mt][s], 0, 0, 0);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                x[mt][s] = __builtin_amdgcn_mfma_f32_16x16x4f32(t.k[s][c][e], qf[mt][c][e], x[mt][s], 0, 0, 0);
            }
          }
    };
    // Scores to probabilities (in x), with the running max and sum.
    auto softmax = [&](unsigned seen, bool whole, int key0) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float top = -INFINITY;
#pragma unroll
        for (int s = 0; s < S::kSubs; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float y = a.rules.template log2_score<!kHalf || kWideCap>(x[mt][s][e]);
            if (a.slopes != nullptr)
              y -= slope[mt] * static_cast<float>(n - 1 - (key0 + 16 * s + 4 * g + e));
            if (!whole) y = (seen >> (4 * s + e)) & 1 ? y : -INFINITY;
            x[mt][s][e] = y;
            top = __builtin_elementwise_maximum(top, y);
          }
        top = opl::max_lane_xor32(opl::combine_xor16_f32<opl::MaxOp>(top));
        const bool moves = kHalf ? top > row_max[mt] + kLazy : top > row_max[mt];
        if (__builtin_amdgcn_ballot_w64(moves) != 0) {
          const float m = fmaxf(row_max[mt], top);
          const float alpha = opl::fast_exp2(row_max[mt] - m);
          row_max[mt] = m;
          sums[mt] *= alpha;
#pragma unroll
          for (int i = 0; i < S::kBlocks; ++i) o[mt][i] *= alpha;
        }
#pragma unroll
        for (int s = 0; s < S::kSubs; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[mt][s][e] = opl::fast_exp2(x[mt][s][e] - row_max[mt] + (kHalf ? kBoost : 0.0f));
      }
    };
    auto values = [&](typename S::Tile& t, unsigned seen, bool whole) {
      if (!whole) {  // values of hidden keys are zeros: 0 x NaN is NaN
#pragma unroll
        for (int j = 0; j < S::kVRows; ++j)
          if (!((seen >> j) & 1)) {
#pragma unroll
            for (int u = 0; u < S::kVC; ++u) t.v[j][u] = typename S::VFrag{};
          }
      }
      if constexpr (kHalf) {
        half8 p[MT], ones;
#pragma unroll
        for (int j = 0; j < 8; ++j) ones[j] = static_cast<_Float16>(1.0f);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int j = 0; j < 8; ++j) p[mt][j] = static_cast<_Float16>(x[mt][j / 4][j % 4]);
          sums[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, p[mt], sums[mt], 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < S::kVC; ++u)
#pragma unroll
          for (int w = 0; w < S::kVW; ++w) {
            half8 f;
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = t.v[j][u][w];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
              o[mt][u * S::kVW + w] =
                  __builtin_amdgcn_mfma_f32_16x16x32_f16(f, p[mt], o[mt][u * S::kVW + w], 0, 0, 0);
          }
      } else {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sums[mt][0] += x[mt][0][e];  // this lane's keys only; joined below
#pragma unroll
            for (int u = 0; u < S::kVC; ++u)
#pragma unroll
              for (int w = 0; w < S::kVW; ++w)
                o[mt][u * S::kVW + w] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                    t.v[e][u][w], x[mt][0][e], o[mt][u * S::kVW + w], 0, 0, 0);
          }
      }
    };

    // ---- the wavefront's tiles: key0, key0 + kUnitKeys, ...
    constexpr unsigned kAll = (1u << (4 * S::kSubs)) - 1;
    int key0 = base_key + wave * S::kKeys;
    if (key0 < last_key) {
      typename S::Tile t;
      Rows rows = rows_of_tile(key0, look_up(key0));
      load_k(t, rows);
      load_v(t, rows);
      Pages next = look_up(key0 + kUnitKeys);
      for (;;) {
        const int key1 = key0 + kUnitKeys;
        const unsigned seen = rows.seen;
        const bool whole = __builtin_amdgcn_ballot_w64(seen != kAll) == 0;
        scores(t);
        __builtin_amdgcn_sched_barrier(0);
        if (key1 < last_key) {
          rows = rows_of_tile(key1, next);
          load_k(t, rows);
          next = look_up(key1 + kUnitKeys);
        }
        __builtin_amdgcn_sched_barrier(0);
        softmax(seen, whole, key0);
        values(t, seen, whole);
        __builtin_amdgcn_sched_barrier(0);
        if (key1 >= last_key) break;
        load_v(t, rows);
        key0 = key1;
      }
    }

    // ---- join the four wavefronts through LDS
    __syncthreads();  // the previous row's readers are done
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float l = sums[mt][0];
      if constexpr (!kHalf) l = opl::sum_lane_xor32(opl::combine_xor16_f32<opl::SumOp>(l));
      float* row = joined[wave][16 * mt + col];
#pragma unroll
      for (int u = 0; u < S::kVC; ++u)
#pragma unroll
        for (int w = 0; w < S::kVW; ++w)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            row[(16 * u + 4 * g + r) * S::kVW + w] = o[mt][u * S::kVW + w][r];
      if (g == 0) {
        row[DP] = row_max[mt];
        row[DP + 1] = l;
      }
    }
    __syncthreads();
    const bool cut = a.direct > 1 || unit != row0 || stop != row0 + units;
    const int slot = a.direct > 0 ? unit : 2 * static_cast<int>(blockIdx.x) + (unit == row0 ? 1 : 0);
    for (int i = threadIdx.x; i < heads * (DP / 4); i += kThreads) {
      const int hh = i / (DP / 4);
      const int d = (i % (DP / 4)) * 4;
      float m = -FLT_MAX;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) m = fmaxf(m, joined[w][hh][DP]);
      float l = 0.0f;
      floatx4 v = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = opl::fast_exp2(joined[w][hh][DP] - m);
        l += f * joined[w][hh][DP + 1];
        v += f * *reinterpret_cast<const floatx4*>(&joined[w][hh][d]);
      }
      if (cut) {
        float* part = a.part + (static_cast<std::int64_t>(slot) * kHeads + hh) * kPitch;
        *reinterpret_cast<floatx4*>(part + d) = v;
        if (d == 0) {
          part[DP] = m;
          part[DP + 1] = l;
        }
      } else if (d < dm) {
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        typedef T Out __attribute__((ext_vector_type(4)));
        Out y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = static_cast<T>(v[e] * inv);
        *reinterpret_cast<Out*>(a.out + (static_cast<std::int64_t>(b) * a.q_heads + head0 + hh) * dm + d) = y;
      }
    }
    // The workgroup in which a cut row starts says where it ends (its last row).
    if (a.cut != nullptr && stop == end && threadIdx.x == 0) {
      // workgroup of unit u: the largest w with w total / G <= u
      const long long last = (static_cast<long long>(row0 + units) * G - 1) / total;
      const bool starts = cut && unit == row0;
      a.cut[2 * blockIdx.x] = starts ? b * rows_of + row_in : -1;
      a.cut[2 * blockIdx.x + 1] = static_cast<int>(last);
    }
    unit = stop;
  }
}

// Adds the pieces of the rows that are in pieces, in order. Direct: a workgroup
// per row and head. Shared-out units: a workgroup per kJoinWaves heads of the row
// that starts in workgroup w of the launch before and ends in a later one; its
// first piece is w's second slot, or the first if w starts with it, the others
// are the first slots of the workgroups after w.
// kWavesPerHead wavefronts take every kWavesPerHead-th piece of a head, a lane
// DP / 64 dims: 1 where rows have few pieces, as there are many rows; all of
// the workgroup's where few rows have many.
constexpr int kJoinWaves = 8;
template <typename T, int DP, int MT, int kWavesPerHead>
__global__ __launch_bounds__(kJoinWaves * opl::kWaveSize) void paged_join_kernel(const PagedArgs<T> a) {
  constexpr int kHeads = 16 * MT;
  constexpr int kPitch = DP + 4;
  constexpr int kDims = DP / opl::kWaveSize;
  constexpr int kPerGroup = kJoinWaves / kWavesPerHead;  // heads of a workgroup
  typedef float Dims __attribute__((ext_vector_type(kDims)));
  __shared__ float top[kJoinWaves], weight[kJoinWaves], joined[kJoinWaves][DP];
  const int rows_of = a.kv_heads * a.tiles_of_heads;
  const int head_groups = (min(kHeads, a.group) + kPerGroup - 1) / kPerGroup;
  const int item = blockIdx.x / head_groups;  // a row, or a workgroup of the launch before
  const int lane = threadIdx.x % opl::kWaveSize;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / opl::kWaveSize);
  const int hh = blockIdx.x % head_groups * kPerGroup + wave / kWavesPerHead;
  int row_id, first, second, step, count;
  if (a.direct > 0) {
    row_id = item;
    first = row_id * a.direct;
    second = first + 1;
    step = 1;
    count = a.direct;
  } else {
    row_id = a.cut[2 * item];
    const int last = a.cut[2 * item + 1];
    if (row_id < 0) return;
    first = 2 * item + 1;
    second = 2 * (item + 1);
    step = 2;
    count = last - item + 1;
  }
  const int b = row_id / rows_of, row_in = row_id % rows_of;
  const int head_tile = row_in % a.tiles_of_heads;
  const bool real = hh < min(kHeads, a.group - head_tile * kHeads);
  float m = -FLT_MAX, l = 0.0f;
  Dims v = {};
  constexpr int kAhead = 8;  // pieces in flight
  for (int j0 = wave % kWavesPerHead; real && j0 < count; j0 += kWavesPerHead * kAhead) {
    float pm[kAhead], pl[kAhead];
    Dims po[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int j = j0 + kWavesPerHead * k;
      const int slot = j == 0 || j >= count ? first : second + (j - 1) * step;
      const float* piece = a.part + (static_cast<std::int64_t>(slot) * kHeads + hh) * kPitch;
      pm[k] = piece[DP];
      pl[k] = piece[DP + 1];
      po[k] = *reinterpret_cast<const Dims*>(piece + kDims * lane);
      if (j >= count) pm[k] = -FLT_MAX, pl[k] = 0.0f;
    }
    float to = m;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) to = fmaxf(to, pm[k]);
    const float f = opl::fast_exp2(m - to);
    m = to;
    l *= f;
    v *= f;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const float w = opl::fast_exp2(pm[k] - m);
      l += w * pl[k];
      // (An empty piece has a sum of 0 and nothing in O.)
      if (pl[k] != 0.0f) v += w * po[k];
    }
  }
  if constexpr (kWavesPerHead > 1) {
    if (lane == 0) {
      top[wave] = m;
      weight[wave] = l;
    }
    *reinterpret_cast<Dims*>(&joined[wave][kDims * lane]) = v;
    __syncthreads();
    if (wave != 0) return;
    static_assert(kWavesPerHead == kJoinWaves, "one head per workgroup");
#pragma unroll
    for (int w = 1; w < kWavesPerHead; ++w) m = fmaxf(m, top[w]);
    l = 0.0f;
    v = Dims{};
#pragma unroll
    for (int w = 0; w < kWavesPerHead; ++w) {
      const float f = opl::fast_exp2(top[w] - m);
      l += f * weight[w];
      v += f * *reinterpret_cast<const Dims*>(&joined[w][kDims * lane]);
    }
  }
  if (!real || kDims * lane >= a.head_dim) return;
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  const int head = (row_in / a.tiles_of_heads) * a.group + head_tile * kHeads + hh;
  T* const out = a.out + (static_cast<std::int64_t>(b) * a.q_heads + head) * a.head_dim + kDims * lane;
#pragma unroll
  for (int e = 0; e < kDims; ++e) out[e] = static_cast<T>(v[e] * inv);
}

// The launch of a call and the scratch it needs.
struct Plan {
  int workgroups;
  int direct;          // units per row with a workgroup each, 0: shared out
  bool join;           // rows can be in pieces
  std::size_t part_bytes, bytes;
};

Plan plan_of(const opl::PagedShape& s, std::size_t element_bytes) {
  const int group = s.q_heads / s.kv_heads;
  const int heads = group > 16 ? 32 : 16;
  const int unit = opl::paged_unit_keys(element_bytes);
  const long long rows =
      static_cast<long long>(s.batch) * s.kv_heads * ((group + opl::kPagedHeads - 1) / opl::kPagedHeads);
  const long long tokens = static_cast<long long>(s.max_pages) * s.page_size;
  const long long row_units = (tokens + unit - 1) / unit;
  Plan p;
  p.direct = rows * row_units <= kDirectUnits ? static_cast<int>(row_units) : 0;
  p.workgroups = static_cast<int>(p.direct ? rows * row_units : kWorkgroups);
  p.join = row_units > 1;
  const int dp = s.head_dim > 64 ? 128 : 64;
  const std::size_t slots = static_cast<std::size_t>(p.workgroups) * (p.direct ? 1 : 2);
  p.part_bytes = p.join ? slots * heads * (dp + 4) * sizeof(float) : 0;
  p.bytes = p.part_bytes +
            (p.join && !p.direct ? static_cast<std::size_t>(p.workgroups) * 2 * sizeof(std::int32_t) : 0);
  return p;
}

template <typename T, int DP, int MT, bool kPaged16, bool kStream>
void start(const PagedArgs<T>& a, dim3 grid, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (a.rules.wide_cap()) {
      paged_attention_kernel<T, DP, MT, kPaged16, kStream, true><<<grid, dim3(kThreads), 0, stream>>>(a);
      return;
    }
  }
  paged_attention_kernel<T, DP, MT, kPaged16, kStream, false><<<grid, dim3(kThreads), 0, stream>>>(a);
}

template <typename T, int DP, int MT>
hipError_t launch(PagedArgs<T> a, const Plan& plan, void* scratch, hipStream_t stream) {
  a.direct = plan.direct;
  a.part = static_cast<float*>(scratch);
  a.cut = plan.join && !plan.direct
              ? reinterpret_cast<std::int32_t*>(static_cast<unsigned char*>(scratch) + plan.part_bytes)
              : nullptr;
  // The cache's bytes, as far as the page table can reach them.
  const std::uint64_t row_bytes = 2ull * a.kv_heads * a.head_dim * sizeof(T);
  const std::uint64_t held = static_cast<std::uint64_t>(a.pages) * a.page_size * row_bytes;
  const std::uint64_t reach = static_cast<std::uint64_t>(a.max_pages) * a.page_size * a.batch * row_bytes;
  const bool stream_past = (held < reach ? held : reach) >= kStreamBytes;
  const dim3 grid(plan.workgroups);
  if (a.page_size % 16 == 0) {
    if (stream_past)
      start<T, DP, MT, true, true>(a, grid, stream);
    else
      start<T, DP, MT, true, false>(a, grid, stream);
  } else {
    if (stream_past)
      start<T, DP, MT, false, true>(a, grid, stream);
    else
      start<T, DP, MT, false, false>(a, grid, stream);
  }
  if (plan.join) {
    const int most = a.group < 16 * MT ? a.group : 16 * MT;
    const unsigned rows = static_cast<unsigned>(a.batch) * a.kv_heads * a.tiles_of_heads;
    const dim3 join_block(kJoinWaves * opl::kWaveSize);
    if (plan.direct)
      paged_join_kernel<T, DP, MT, kJoinWaves><<<dim3(rows * most), join_block, 0, stream>>>(a);
    else if (rows < kFewRows)
      paged_join_kernel<T, DP, MT, kJoinWaves><<<dim3(plan.workgroups * most), join_block, 0, stream>>>(a);
    else
      paged_join_kernel<T, DP, MT, 1>
          <<<dim3(plan.workgroups * ((most + kJoinWaves - 1) / kJoinWaves)), join_block, 0, stream>>>(a);
  }
  return hipGetLastError();
}

template <typename T>
int paged_entry(PagedArgs<T> a, float scale, float softcap, const opl::ScratchSource& src,
                void* stream_handle) {
  const opl::PagedShape shape = {a.batch,    a.q_heads,   a.kv_heads,
                                 a.head_dim, a.page_size, a.max_pages};
  if (a.q == nullptr || a.key_cache == nullptr || a.value_cache == nullptr ||
      a.page_table == nullptr || a.lengths == nullptr || a.out == nullptr ||
      !opl::paged_shape_ok(shape, sizeof(T)) ||
      !opl::paged_cache_ok(a.pages, a.kv_heads, a.page_size) ||
      !opl::score_rules_ok(scale, a.window, softcap) ||
      a.q_stride < static_cast<std::int64_t>(a.q_heads) * a.head_dim ||
      a.table_stride < a.max_pages || !opl::aligned_rows(a.q, sizeof(T), a.q_stride) ||
      !opl::aligned16(a.key_cache) || !opl::aligned16(a.value_cache) || !opl::aligned16(a.out))
    return hipErrorInvalidValue;
  a.group = a.q_heads / a.kv_heads;
  a.tiles_of_heads = (a.group + opl::kPagedHeads - 1) / opl::kPagedHeads;
  a.rules = opl::ScoreRules::of(scale, softcap);
  a.page_of = opl::Divider::by(a.page_size);
  const Plan plan = plan_of(shape, sizeof(T));
  if (src.workspace_mode ? !opl::workspace_ok(src.data, src.bytes, plan.bytes)
                         : plan.bytes > opl::kArenaBytes)
    return hipErrorInvalidValue;
  const hipStream_t stream = static_cast<hipStream_t>(stream_handle);
  auto run = [&](void* scratch) {
    if (a.head_dim > 64)
      return a.group > 16 ? launch<T, 128, 2>(a, plan, scratch, stream)
                          : launch<T, 128, 1>(a, plan, scratch, stream);
    return a.group > 16 ? launch<T, 64, 2>(a, plan, scratch, stream)
                        : launch<T, 64, 1>(a, plan, scratch, stream);
  };
  if (plan.bytes == 0) return run(nullptr);
  opl::ScratchLease lease(stream, src.workspace_mode ? src.data : nullptr, src.bytes);
  if (lease.status() != hipSuccess) return lease.status();
  return run(lease.data());
}

template <typename T>
std::size_t paged_workspace(const opl::PagedShape& s) {
  return opl::paged_shape_ok(s, sizeof(T)) ? plan_of(s, sizeof(T)).bytes : 0;
}

template <typename T, typename U>
PagedArgs<T> args_of(const U* q, std::int64_t q_stride, const U* key_cache, const U* value_cache,
                     const std::int32_t* page_table, std::int64_t table_stride,
                     const std::int32_t* lengths, const float* slopes, U* output, int batch,
                     int q_heads, int kv_heads, int head_dim, int pages, int page_size,
                     int max_pages, int window) {
  PagedArgs<T> a = {};
  a.q = reinterpret_cast<const T*>(q);
  a.key_cache = reinterpret_cast<const T*>(key_cache);
  a.value_cache = reinterpret_cast<const T*>(value_cache);
  a.page_table = page_table;
  a.lengths = lengths;
  a.slopes = slopes;
  a.out = reinterpret_cast<T*>(output);
  a.q_stride = q_stride;
  a.table_stride = table_stride;
  a.batch = batch;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.head_dim = head_dim;
  a.pages = pages;
  a.page_size = page_size;
  a.max_pages = max_pages;
  a.window = window;
  return a;
}

}  // namespace

#define OPL_PAGED_ENTRIES(NAME, U, T)                                                             \
  extern "C" size_t operatorlib_paged_attention_##NAME##_workspace_size(                          \
      int batch, int q_heads, int kv_heads, int head_dim, int page_size, int max_pages) {         \
    return paged_workspace<T>({batch, q_heads, kv_heads, head_dim, page_size, max_pages});        \
  }                                                                                               \
  extern "C" int operatorlib_paged_attention_##NAME##_ws(                                         \
      const U* q, int64_t q_stride, const U* key_cache, const U* value_cache,                     \
      const int32_t* page_table, int64_t table_stride, const int32_t* lengths,                    \
      const float* slopes, U* output, int batch, int q_heads, int kv_heads, int head_dim,         \
      int pages, int page_size, int max_pages, float scale, int window, float softcap,            \
      void* workspace, size_t workspace_bytes, void* stream) {                                    \
    return paged_entry<T>(                                                                        \
        args_of<T>(q, q_stride, key_cache, value_cache, page_table, table_stride, lengths,        \
                   slopes, output, batch, q_heads, kv_heads, head_dim, pages, page_size,          \
                   max_pages, window),                                                            \
        scale, softcap, opl::ScratchSource{true, workspace, workspace_bytes}, stream);            \
  }                                                                                               \
  extern "C" int operatorlib_paged_attention_##NAME(                                              \
      const U* q, int64_t q_stride, const U* key_cache, const U* value_cache,                     \
      const int32_t* page_table, int64_t table_stride, const int32_t* lengths,                    \
      const float* slopes, U* output, int batch, int q_heads, int kv_heads, int head_dim,         \
      int pages, int page_size, int max_pages, float scale, int window, float softcap,            \
      void* stream) {                                                                             \
    return paged_entry<T>(                                                                        \
        args_of<T>(q, q_stride, key_cache, value_cache, page_table, table_stride, lengths,        \
                   slopes, output, batch, q_heads, kv_heads, head_dim, pages, page_size,          \
                   max_pages, window),                                                            \
        scale, softcap, opl::ScratchSource{}, stream);                                            \
  }

OPL_PAGED_ENTRIES(f16, operatorlib_half_t, _Float16)
OPL_PAGED_ENTRIES(f32, float, float)
