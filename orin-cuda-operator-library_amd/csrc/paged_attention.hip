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
// is bound by reading the cache. A wavefront loads tile i + 1 while it
// computes tile i (16 KiB in flight per wavefront, 8 wavefronts per CU).
//
// Work split. The host does not know the lengths. The unit of work is four
// tiles (one per wavefront of a workgroup) of one (sequence, key head); the
// units of all of them form one line, and workgroup w of G takes an equal,
// contiguous piece of it, whatever mix of long and short sequences it holds.
// Every workgroup finds its piece from the lengths (a scan of at most a few
// of them per thread). A row (sequence, key head) that lies in one piece is
// written at once; one cut by piece borders leaves an unnormalised O with its
// max and sum per piece, and paged_join_kernel adds them in order of the
// workgroups (deterministic). A piece cuts at most its first and its last
// row: two slots of scratch per workgroup.

#include <hip/hip_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "common.hpp"
#include "lm_validate.hpp"
#include "operatorlib/lm_c.h"
#include "scores.hpp"
#include "scratch.hpp"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = 4;
// Workgroups of a launch: two per CU of an MI355X.
constexpr int kWorkgroups = 512;
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
  float* part;          // [workgroups][2][heads of a row][DP + 4]: O, max, sum
  std::int32_t* cut;    // [rows][2]: slot of the first piece and the last workgroup
                        // of a cut row; (0, -1) of any other
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

// MT: 16-head operands per workgroup (group up to 16 MT). kPaged16: pages hold
// whole 16-key blocks, so that a block's rows follow each other.
template <typename T, int DP, int MT, bool kPaged16>
__global__ __launch_bounds__(kThreads) void paged_attention_kernel(const PagedArgs<T> a) {
  using S = Shape<T, DP>;
  constexpr bool kHalf = S::kHalf;
  constexpr int kHeads = 16 * MT;
  constexpr int kUnitKeys = kWaves * S::kKeys;
  constexpr int kPitch = DP + 4;  // floats of a head's row in LDS: rows 16 bytes apart in the banks
  __shared__ __attribute__((aligned(16))) float joined[kWaves][kHeads][kPitch];
  __shared__ int scan[kWaves];
  __shared__ int found[4];

  const int lane = threadIdx.x % opl::kWaveSize;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / opl::kWaveSize);
  const int col = lane % 16;
  const int g = lane / 16;
  const int rows_of = a.kv_heads * a.tiles_of_heads;  // rows of a sequence

  // ---- this workgroup's piece of the units --------------------------------
  const int chunk = (a.batch + kThreads - 1) / kThreads;
  const int b_first = min(a.batch, static_cast<int>(threadIdx.x) * chunk);
  const int b_last = min(a.batch, b_first + chunk);
  int mine = 0;
  for (int b = b_first; b < b_last; ++b) mine += units_of<kUnitKeys>(key_range(a, b)) * rows_of;
  int upto = mine;  // inclusive scan over the wavefront, then over the four
#pragma unroll
  for (int step = 1; step < opl::kWaveSize; step *= 2) {
    const int below = __shfl_up(upto, step);
    if (lane >= step) upto += below;
  }
  if (lane == opl::kWaveSize - 1) scan[wave] = upto;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) upto += scan[w];
    total += scan[w];
  }
  // (No more pieces than units: each of a cut row's workgroups has a part of it.)
  const long long G = min(static_cast<int>(gridDim.x), total);
  if (blockIdx.x >= G) return;
  const int begin = static_cast<int>(static_cast<long long>(blockIdx.x) * total / G);
  const int end = static_cast<int>((static_cast<long long>(blockIdx.x) + 1) * total / G);
  if (begin >= upto - mine && begin < upto) {
    int at = upto - mine, b = b_first;
    for (;; ++b) {
      const int u = units_of<kUnitKeys>(key_range(a, b)) * rows_of;
      if (begin < at + u) break;
      at += u;
    }
    found[0] = b;
    found[1] = at;
  }
  __syncthreads();
  int b = __builtin_amdgcn_readfirstlane(found[0]);
  int at = __builtin_amdgcn_readfirstlane(found[1]);  // first unit of sequence b
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

  int unit = begin;
  while (unit < end) {
    // ---- the row (sequence b, key head, tile of heads) that `unit` lies in
    int2 range = key_range(a, b);
    int units = units_of<kUnitKeys>(range);
    while (unit >= at + units * rows_of) {
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
    // Page of token `key` (< n), or -1 if it is not a page.
    auto page_of = [&](int key) {
      const int p = table[key / a.page_size];
      return p >= 0 && p < a.pages ? p : -1;
    };
    // First element of a cache row.
    auto row_start = [&](int page, int key) {
      return (static_cast<std::int64_t>(page) * a.kv_heads + kv_head) * a.page_size +
             key % a.page_size;
    };

    // Cache rows of the lane's K and V rows in the tile from key0, and which
    // of the lane's keys are visible (bit 4 s + r: key 16 s + 4 g + r).
    // Rows of hidden keys are those of cache row 0.
    struct Rows {
      std::int64_t sub[S::kSubs];            // kPaged16: first row of each block
      std::int64_t k[S::kSubs];              // else: the lane's K rows
      std::int64_t v[kPaged16 ? 1 : S::kVRows];
      unsigned seen;
    };
    auto rows_at = [&](int key0) {
      Rows r;
      r.seen = 0;
      if constexpr (kPaged16) {
#pragma unroll
        for (int s = 0; s < S::kSubs; ++s) {
          const int key = key0 + 16 * s;
          const int page = key < n ? __builtin_amdgcn_readfirstlane(page_of(key)) : -1;
          r.sub[s] = page >= 0 ? row_start(page, key) : 0;
          if (page >= 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int mk = key + 4 * g + e;
              if (mk >= lo && mk < n) r.seen |= 1u << (4 * s + e);
            }
          }
        }
      } else {
#pragma unroll
        for (int s = 0; s < S::kSubs; ++s) {
          const int key = key0 + 16 * s + col;
          const int page = key < n ? page_of(key) : -1;
          r.k[s] = page >= 0 ? row_start(page, key) : 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int from = 4 * g + e;  // the lane that looked up key 16 s + 4 g + e
            const int mk = key0 + 16 * s + from;
            r.v[4 * s + e] = __shfl(r.k[s], from);
            if (__shfl(page, from) >= 0 && mk >= lo && mk < n) r.seen |= 1u << (4 * s + e);
          }
        }
      }
      return r;
    };
    auto load = [&](typename S::Tile& t, const Rows& r) {
#pragma unroll
      for (int s = 0; s < S::kSubs; ++s) {
        const T* base = kPaged16 ? a.key_cache + r.sub[s] * dm + col * dm : a.key_cache + r.k[s] * dm;
#pragma unroll
        for (int c = 0; c < S::kSteps; ++c)
          t.k[s][c] = *reinterpret_cast<const typename S::KFrag*>(base + k_dim[c]);
      }
#pragma unroll
      for (int j = 0; j < S::kVRows; ++j) {
        const T* base = kPaged16 ? a.value_cache + r.sub[j / 4] * dm + (4 * g + j % 4) * dm
                                 : a.value_cache + r.v[kPaged16 ? 0 : j] * dm;
#pragma unroll
        for (int u = 0; u < S::kVC; ++u)
          t.v[j][u] = *reinterpret_cast<const typename S::VFrag*>(base + v_dim[u]);
      }
    };
    auto compute = [&](typename S::Tile& t, unsigned seen, int key0) {
      constexpr unsigned kAll = (1u << (4 * S::kSubs)) - 1;
      const bool whole = __builtin_amdgcn_ballot_w64(seen != kAll) == 0;
      if (!whole) {  // values of hidden keys are zeros: 0 x NaN is NaN
#pragma unroll
        for (int j = 0; j < S::kVRows; ++j)
          if (!((seen >> j) & 1)) {
#pragma unroll
            for (int u = 0; u < S::kVC; ++u) t.v[j][u] = typename S::VFrag{};
          }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        floatx4 x[S::kSubs];
#pragma unroll
        for (int s = 0; s < S::kSubs; ++s) x[s] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < S::kSteps; ++c)
#pragma unroll
          for (int s = 0; s < S::kSubs; ++s) {
            if constexpr (kHalf) {
              x[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(t.k[s][c], qf[mt][c], x[s], 0, 0, 0);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                x[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(t.k[s][c][e], qf[mt][c][e], x[s], 0, 0, 0);
            }
          }
        float top = -INFINITY;
#pragma unroll
        for (int s = 0; s < S::kSubs; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float y = a.rules.template log2_score<!kHalf>(x[s][e]);
            if (a.slopes != nullptr)
              y -= slope[mt] * static_cast<float>(n - 1 - (key0 + 16 * s + 4 * g + e));
            if (!whole && !((seen >> (4 * s + e)) & 1)) y = -INFINITY;
            x[s][e] = y;
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
        if constexpr (kHalf) {
          half8 p;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            p[j] = static_cast<_Float16>(opl::fast_exp2(x[j / 4][j % 4] - row_max[mt] + kBoost));
          half8 ones;
#pragma unroll
          for (int j = 0; j < 8; ++j) ones[j] = static_cast<_Float16>(1.0f);
          sums[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, p, sums[mt], 0, 0, 0);
#pragma unroll
          for (int u = 0; u < S::kVC; ++u)
#pragma unroll
            for (int w = 0; w < S::kVW; ++w) {
              half8 f;
#pragma unroll
              for (int j = 0; j < 8; ++j) f[j] = t.v[j][u][w];
              o[mt][u * S::kVW + w] =
                  __builtin_amdgcn_mfma_f32_16x16x32_f16(f, p, o[mt][u * S::kVW + w], 0, 0, 0);
            }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = opl::fast_exp2(x[0][e] - row_max[mt]);
            sums[mt][0] += p;  // this lane's keys only; joined below
#pragma unroll
            for (int u = 0; u < S::kVC; ++u)
#pragma unroll
              for (int w = 0; w < S::kVW; ++w)
                o[mt][u * S::kVW + w] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                    t.v[e][u][w], p, o[mt][u * S::kVW + w], 0, 0, 0);
          }
        }
      }
    };

    // ---- the wavefront's tiles: key0, key0 + kUnitKeys, ...
    int key0 = base_key + wave * S::kKeys;
    if (key0 < last_key) {
      typename S::Tile ta, tb;
      Rows ra = rows_at(key0), rb;
      load(ta, ra);
      for (;;) {
        const int key1 = key0 + kUnitKeys;
        const bool more = key1 < last_key;
        if (more) {
          rb = rows_at(key1);
          load(tb, rb);
        }
        compute(ta, ra.seen, key0);
        if (!more) break;
        key0 = key1 + kUnitKeys;
        const bool again = key0 < last_key;
        if (again) {
          ra = rows_at(key0);
          load(ta, ra);
        }
        compute(tb, rb.seen, key1);
        if (!again) break;
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
    const bool cut = unit != row0 || stop != row0 + units;
    const int slot = row0 <= begin ? 0 : 1;
    const int row_id = b * rows_of + row_in;
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
        float* part = a.part + ((static_cast<std::int64_t>(blockIdx.x) * 2 + slot) * kHeads + hh) * kPitch;
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
    // The workgroup that starts a row says who has its pieces.
    if (a.cut != nullptr && unit == row0 && threadIdx.x == 0) {
      // workgroup of unit u: the largest w with w total / G <= u
      const long long last = (static_cast<long long>(row0 + units) * G - 1) / total;
      a.cut[2 * row_id] = 2 * static_cast<int>(blockIdx.x) + slot;
      a.cut[2 * row_id + 1] = cut ? static_cast<int>(last) : -1;
    }
    unit = stop;
  }
}

// Adds the pieces of a cut row, in order: one workgroup per row. The first
// piece is in either slot of its workgroup, the others in the first slot of
// the workgroups after it (which start with this row).
template <typename T, int DP, int MT>
__global__ __launch_bounds__(kThreads) void paged_join_kernel(const PagedArgs<T> a) {
  constexpr int kHeads = 16 * MT;
  constexpr int kPitch = DP + 4;
  const int row_id = blockIdx.x;
  const int first = a.cut[2 * row_id];
  const int more = a.cut[2 * row_id + 1] - first / 2;  // pieces after the first
  if (a.cut[2 * row_id + 1] < 0) return;
  const int rows_of = a.kv_heads * a.tiles_of_heads;
  const int b = row_id / rows_of, row_in = row_id % rows_of;
  const int head_tile = row_in % a.tiles_of_heads;
  const int heads = min(kHeads, a.group - head_tile * kHeads);
  const int head0 = (row_in / a.tiles_of_heads) * a.group + head_tile * kHeads;
  for (int i = threadIdx.x; i < heads * (DP / 4); i += kThreads) {
    const int hh = i / (DP / 4);
    const int d = (i % (DP / 4)) * 4;
    if (d >= a.head_dim) continue;
    const float* piece = a.part + (static_cast<std::int64_t>(first) * kHeads + hh) * kPitch;
    const float* next =
        a.part + (static_cast<std::int64_t>(first / 2 + 1) * 2 * kHeads + hh) * kPitch;
    float m = piece[DP];
    for (int j = 0; j < more; ++j) m = fmaxf(m, next[j * 2 * kHeads * kPitch + DP]);
    float f = opl::fast_exp2(piece[DP] - m);
    float l = f * piece[DP + 1];
    floatx4 v = f * *reinterpret_cast<const floatx4*>(piece + d);
#pragma unroll 4
    for (int j = 0; j < more; ++j) {
      const float* p = next + j * 2 * kHeads * kPitch;
      f = opl::fast_exp2(p[DP] - m);
      l += f * p[DP + 1];
      v += f * *reinterpret_cast<const floatx4*>(p + d);
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    typedef T Out __attribute__((ext_vector_type(4)));
    Out y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = static_cast<T>(v[e] * inv);
    *reinterpret_cast<Out*>(a.out + (static_cast<std::int64_t>(b) * a.q_heads + head0 + hh) *
                                        a.head_dim + d) = y;
  }
}

// The launch of a call and the scratch it needs.
struct Plan {
  int workgroups;
  bool join;           // rows can be cut
  std::size_t part_bytes, bytes;
};

Plan plan_of(const opl::PagedShape& s, std::size_t element_bytes) {
  const int group = s.q_heads / s.kv_heads;
  const int heads = group > 16 ? 32 : 16;
  const int unit = opl::paged_unit_keys(element_bytes);
  const long long rows =
      static_cast<long long>(s.batch) * s.kv_heads * ((group + opl::kPagedHeads - 1) / opl::kPagedHeads);
  const long long tokens = static_cast<long long>(s.max_pages) * s.page_size;
  const long long units = rows * ((tokens + unit - 1) / unit);
  Plan p;
  p.workgroups = static_cast<int>(units < kWorkgroups ? units : kWorkgroups);
  p.join = tokens > unit;
  const int dp = s.head_dim > 64 ? 128 : 64;
  p.part_bytes = p.join ? static_cast<std::size_t>(p.workgroups) * 2 * heads * (dp + 4) * sizeof(float) : 0;
  p.bytes = p.join ? p.part_bytes + static_cast<std::size_t>(rows) * 2 * sizeof(std::int32_t) : 0;
  return p;
}

template <typename T, int DP, int MT>
hipError_t launch(PagedArgs<T> a, const Plan& plan, void* scratch, hipStream_t stream) {
  const dim3 block(kThreads);
  a.part = static_cast<float*>(scratch);
  a.cut = plan.join ? reinterpret_cast<std::int32_t*>(static_cast<unsigned char*>(scratch) + plan.part_bytes)
                    : nullptr;
  if (a.page_size % 16 == 0)
    paged_attention_kernel<T, DP, MT, true><<<dim3(plan.workgroups), block, 0, stream>>>(a);
  else
    paged_attention_kernel<T, DP, MT, false><<<dim3(plan.workgroups), block, 0, stream>>>(a);
  if (plan.join) {
    const unsigned rows = static_cast<unsigned>(a.batch) * a.kv_heads * a.tiles_of_heads;
    paged_join_kernel<T, DP, MT><<<dim3(rows), block, 0, stream>>>(a);
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
