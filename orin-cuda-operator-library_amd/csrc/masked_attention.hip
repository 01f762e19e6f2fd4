// masked_attention: the tokens of a prompt attend to each other, with the
// masks and score rules of language models (operatorlib/lm_c.h).
//
// Per (batch, query head) the online recurrence of the flash kernels:
// m' = max(m, x), O^T' = O^T 2^(m - m') + V^T P^T, no S x S matrix. The tiles
// and lane layout are attention.hip's: S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_16x16x32_f16 (fp32: 16x16x4), so that the S^T accumulators of a
// lane are its part of the P^T operand; K and V tiles copied global -> LDS by
// buffer loads with the lds modifier, two stages, 16-byte chunks XOR-swizzled;
// V^T read with ds_read_b64_tr_b16; fp16 row sums on the matrix cores; the
// running max moves only by more than kLazyLog2.
//
// What the rules add:
//   * Visibility of key j to query i, without documents, is j < prefix or
//     lo(i) <= j <= hi(i): two compares. lo and hi come from causal and window.
//   * A query block visits the key tiles of the prefix and of
//     [lo(first row), hi(last row)] only. With documents it first marks, per
//     wavefront and 64 keys, whether their span of documents meets that of the
//     wavefront's rows, and whether all of them and all rows are one
//     document: tiles that no wavefront marks are not copied, a wavefront skips
//     those it has not marked, and tiles of one document inside the bounds need
//     no mask. The tiles' ids are copied to LDS with the tiles.
//   * A wavefront applies the mask only in tiles that some of its rows see in
//     part: a branch around the mask alone. (One loop body for both kinds of
//     tile; two bodies made the compiler keep O twice and spill 139 registers.)
//   * A hidden key's probability is 0, but 0 x infinity is NaN: if a block's O
//     ends with a NaN, the block runs again with the non-finite values of V
//     taken for zeros, and then adds them to the rows that see their keys.
//     Blocks without a NaN pay one test.
//
// Measured on MI355X, fp16, 32 + 8 heads of 128:
//   * 8192 tokens, causal: 523 us, 1050 TFLOP/s of the visible products (a large
//     library product runs at 1189): matrix cores and exponentials hardly overlap, as in
//     attention.hip. Capped 612 to 631 us (870 to 900 TFLOP/s), biased 590: bound by the
//     vector units, with three transcendental instructions a capped score.
//   * 11 documents in 8000 tokens: 151 us where the products alone take 67. A
//     workgroup of 10 tiles spends 11 k of its 69 k cycles before the first one (marks
//     5.8 k, queries, first copy) and 3 k behind the last, partial tiles cost a quarter
//     more than whole ones, and the last heavy blocks run when the others are done
//     (a tenth of the workgroups in the last 22 us).

#include <hip/hip_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "attention_tiles.hpp"
#include "common.hpp"
#include "lm_validate.hpp"
#include "operatorlib/lm_c.h"
#include "scores.hpp"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
#define OPL_LDS __attribute__((address_space(3)))

constexpr int kXcds = 8;
constexpr int kRowsPerWave = 32;
// Headroom (log2 units) the running max may lag the true max by.
constexpr float kLazyLog2 = 8.0f;
// Workgroup slots of an XCD that a causal launch balances (attention.hip).
constexpr int kCausalGroupSlots = 64;
// Marks: a bit per 64 keys, up to 2^18 keys; tiles behind those are visited and
// masked whatever their documents.
constexpr int kMarkWords = 128;
constexpr int kIdBytes = 256;  // ids of a tile's keys in LDS, as one wavefront copies them

template <typename T>
struct MaskedArgs {
  const T* q;
  const T* k;
  const T* v;
  T* out;
  opl::MaskedStrides qs, ks, vs, os;
  const float* slopes;
  const std::int32_t* documents;
  const std::int32_t* prefixes;
  int bh, q_heads, group, S, dm, causal, window;
  opl::ScoreRules rules;
};

// What becomes of the scores. kBoth: capped in the precise form, and biased if
// there are slopes; it takes fp16's caps past kSigmaCap too.
enum Rules { kScaled, kCapped, kBiased, kBoth };

template <typename T, int D, int kGroups, int kW, int kTileKeys>
constexpr int kMinWavesPerSimd =
    2 * kGroups * opl::Layout<T, D, kTileKeys>::kStage > 80 * 1024 && kGroups * kW == 4 ? 1 : 2;

// kW wavefronts of 32 query rows share the tiles of a group; kGroups groups
// (small grids) take every kGroups-th tile of the same rows and join at the
// end.
// D: the LDS rows' dims; Dc: those computed (head dims of 65 to 96 take 96 of 128).
template <typename T, int D, int Dc, int kGroups, int kW, int kTileKeys, Rules kRules>
__global__ __launch_bounds__(kW * opl::kWaveSize * kGroups)
__attribute__((amdgpu_waves_per_eu(kMinWavesPerSimd<T, D, kGroups, kW, kTileKeys>, 2)))
void masked_attention_kernel(const MaskedArgs<T> a) {
  using L = opl::Layout<T, D, kTileKeys, Dc>;
  constexpr bool kHalf = L::kSize == 2;
  constexpr bool kCaps = kRules == kCapped || kRules == kBoth;
  constexpr bool kBiases = kRules == kBiased || kRules == kBoth;
  constexpr bool kPrecise = !kHalf || kRules == kBoth;  // (how a score is capped)
  using Frag = typename std::conditional<kHalf, half8, floatx4>::type;
  constexpr int kRows = kW * kRowsPerWave;
  constexpr int kThreads = kW * kGroups * opl::kWaveSize;
  constexpr int kCopies = L::kTile / 16 / (kW * opl::kWaveSize);
  constexpr int kArray = kGroups * L::kStage;
  __shared__ __attribute__((aligned(1024))) unsigned char stage0[kArray];
  __shared__ __attribute__((aligned(1024))) unsigned char stage1[kArray];
  __shared__ __attribute__((aligned(16))) int ids0[kGroups * kIdBytes / 4];
  __shared__ __attribute__((aligned(16))) int ids1[kGroups * kIdBytes / 4];
  __shared__ unsigned marked[kMarkWords];     // some wavefront's bit is set
  __shared__ unsigned some[kW][kMarkWords];   // the documents of the 64 keys and its rows may meet
  __shared__ unsigned single[kW][kMarkWords]; // its rows and the 64 keys are one document
  __shared__ int span[kW][3];                 // least and greatest document of its rows, 1 if it has one
  __shared__ float2 ends[kGroups > 1 ? kGroups * kW : 1][kRowsPerWave];  // max and sum of a row
  __shared__ bool poisoned[kGroups * kW];

  // ---- which rows of which head: XCD x takes a contiguous range of the work,
  // heads in order (the query heads of a key head follow each other), heaviest
  // block of a causal head first, groups of heads interleaved where a head has
  // few blocks (attention.hip).
  const int S = a.S;
  const int q_blocks = (S + kRows - 1) / kRows;
  const int total = q_blocks * a.bh;
  const int per_xcd = (total + kXcds - 1) / kXcds;
  const int w = static_cast<int>(blockIdx.x % kXcds) * per_xcd + static_cast<int>(blockIdx.x / kXcds);
  if (w >= total) return;
  int bh = w / q_blocks;
  int qb = q_blocks - 1 - w % q_blocks;
  if (a.causal || a.documents != nullptr) {
    // Heads whose blocks are taken together: about the slots of an XCD, all of the
    // XCD's where its work is two rounds or less, or with documents, whose heavy
    // blocks are anywhere (11 documents in 8000 tokens, 32 heads: 178 -> 153 us; 3 in
    // 2000 of a batch of 4, every key of a document visible: 191 -> 159).
    const bool all = a.documents != nullptr || per_xcd <= 2 * kCausalGroupSlots;
    const int g = max(1, (all ? per_xcd : kCausalGroupSlots) / q_blocks);
    if (g > 1) {
      const int first = w / (g * q_blocks) * g;
      const int heads = min(g, a.bh - first);
      const int r = w - first * q_blocks;
      bh = first + r % heads;
      qb = q_blocks - 1 - r / heads;
    }
  }
  const int batch = bh / a.q_heads;
  const int head = bh % a.q_heads;
  const int q0 = qb * kRows;
  const int lane = threadIdx.x % opl::kWaveSize;
  const int wave = (threadIdx.x / opl::kWaveSize) % kW;
  const int group = kGroups == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / opl::kWaveSize / kW);
  unsigned char* const st0 = stage0 + group * L::kStage;
  unsigned char* const st1 = stage1 + group * L::kStage;
  int* const id0 = ids0 + group * (kIdBytes / 4);
  int* const id1 = ids1 + group * (kIdBytes / 4);
  const int col = lane % 16;
  const int quad = lane / 16;
  const int wave_row0 = q0 + wave * kRowsPerWave;
  const int dm = a.dm;
  const T* qh = a.q + batch * a.qs.batch + head * a.qs.head;
  const T* kh = a.k + batch * a.ks.batch + (head / a.group) * a.ks.head;
  const T* vh = a.v + batch * a.vs.batch + (head / a.group) * a.vs.head;
  const std::int32_t* docs =
      a.documents != nullptr ? a.documents + static_cast<std::int64_t>(batch) * S : nullptr;
  const int prefix = a.prefixes != nullptr ? min(max(a.prefixes[batch], 0), S) : 0;
  // Bounds of the keys that row i sees outside the prefix. (window up to
  // 2^31 - 1: i - window + 1 cannot underflow, and the sum is taken against S - i.)
  auto low = [&](int i) { return a.window > 0 ? max(0, i - a.window + 1) : 0; };
  auto high = [&](int i) {
    if (a.causal) return min(i, S - 1);
    return a.window > 0 && a.window < S - i ? i + a.window - 1 : S - 1;
  };

  // ---- Q^T operand. (Nothing is done to it on arrival: the reads of documents and
  // the first tile are issued behind it.)
  constexpr int kNoData = static_cast<int>(0x80000000u);
  Frag qf[2][L::kSteps];
  int row_doc[2] = {0, 0};  // without documents every key's id is read as 0
  auto read_q = [&] {
#pragma unroll
    for (int qc = 0; qc < 2; ++qc) {
      const int row = min(wave_row0 + 16 * qc + col, S - 1) * static_cast<int>(a.qs.token);
      const unsigned bytes = static_cast<unsigned>((S - 1) * a.qs.token + dm) * L::kSize;
#pragma unroll
      for (int c = 0; c < L::kSteps; ++c) {
        const int dim = L::kSubK * c + L::kElems * quad;
        const auto x = opl::buffer_load16(qh, bytes, dim < dm ? (row + dim) * L::kSize : kNoData);
        qf[qc][c] = __builtin_bit_cast(Frag, x);
      }
    }
  };
  if (docs == nullptr) read_q();

  // ---- the tiles that the block visits
  const int last_row = min(q0 + kRows, S) - 1;
  const int prefix_tiles = (prefix + kTileKeys - 1) / kTileKeys;
  const int from_tile = low(q0) / kTileKeys;
  const int end_tile = max(prefix_tiles, high(last_row) / kTileKeys + 1);
  if (docs != nullptr) {
    // Lane l of a wavefront takes the 64 keys of chunk c0 + l: their least and
    // greatest id. (A ballot per chunk, one key per lane, took 3.7 us of each
    // workgroup at 8000 keys; a chunk per 16 lanes was no faster than this.)
    struct Ids {
      unsigned least_id;  // of the ids >= 0 (a negative one is a large unsigned)
      int most_id, any_id;
    };
    auto ids_of = [&](int chunk) {
      typedef int Four __attribute__((ext_vector_type(4), aligned(4)));
      Ids r = {0xffffffffu, -1, 0x7fffffff};
      auto take = [&](int id) {
        r.least_id = min(r.least_id, static_cast<unsigned>(id));
        r.most_id = max(r.most_id, id);
        r.any_id = min(r.any_id, id);
      };
      const int first = chunk * 64;
      if (first + 64 <= S) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const Four id = *reinterpret_cast<const Four*>(docs + first + 4 * i);
#pragma unroll
          for (int e = 0; e < 4; ++e) take(id[e]);
        }
      } else {
        for (int key = first; key < first + 64; ++key) take(key < S ? docs[key] : -1);
      }
      return r;
    };
    // Each wavefront of rows: the least and greatest id, by 32 of its lanes.
    const int i = wave_row0 + lane % kRowsPerWave;
    const int id = docs[min(i, S - 1)];
    // The first step's keys are read before the rows' ids are awaited.
    const int chunks = min((end_tile * kTileKeys + 63) / 64, kMarkWords * 32);
    int c0 = threadIdx.x / opl::kWaveSize * 64;
    Ids keys = ids_of(min(c0 + lane, chunks - 1));
    read_q();
    int least_row = i < S && id >= 0 ? id : 0x7fffffff, most_row = i < S ? max(id, -1) : -1;
#pragma unroll
    for (int step = 1; step < kRowsPerWave; step *= 2) {
      least_row = min(least_row, __shfl_xor(least_row, step));
      most_row = max(most_row, __shfl_xor(most_row, step));
    }
#pragma unroll
    for (int qc = 0; qc < 2; ++qc)
      row_doc[qc] = __shfl(id >= 0 ? id : -2, 16 * qc + col);  // (-2: no key's id)
    const bool padded = __builtin_amdgcn_ballot_w64(i < S && id < 0) != 0;
    if (group == 0 && lane == 0) {
      span[wave][0] = least_row;
      span[wave][1] = most_row;
      span[wave][2] = !padded && least_row == most_row;
    }
    __syncthreads();
    for (; c0 < chunks; c0 += kThreads) {
      std::uint64_t any = 0;
#pragma unroll
      for (int r = 0; r < kW; ++r) {
        const int least = span[r][0], most = span[r][1];
        const std::uint64_t within = __builtin_amdgcn_ballot_w64(
            (most >= 0) & (keys.least_id <= static_cast<unsigned>(most)) & (keys.most_id >= least));
        const std::uint64_t same = __builtin_amdgcn_ballot_w64(
            (span[r][2] != 0) & (keys.any_id == least) & (keys.most_id == least));
        any |= within;
        if (lane < 2) {
          some[r][c0 / 32 + lane] = static_cast<unsigned>(within >> (32 * lane));
          single[r][c0 / 32 + lane] = static_cast<unsigned>(same >> (32 * lane));
        }
      }
      if (lane < 2) marked[c0 / 32 + lane] = static_cast<unsigned>(any >> (32 * lane));
      if (c0 + kThreads < chunks) keys = ids_of(min(c0 + kThreads + lane, chunks - 1));
    }
    __syncthreads();
  }
  // The first visited tile from t on (end_tile: none left). Wave-uniform.
  auto visit = [&](int t) {
    if (t >= prefix_tiles && t < from_tile) t = from_tile;
    if (docs != nullptr) {
      while (t < end_tile) {
        const int bit = t * kTileKeys / 64;
        if (bit >= kMarkWords * 32) break;
        const unsigned rest = __builtin_amdgcn_readfirstlane(marked[bit / 32]) >> (bit % 32);
        if (rest & 1) break;
        // the next marked 64 keys of this word, or the next word
        const int skip = rest != 0 ? __builtin_ctz(rest) : 32 - bit % 32;
        t = (bit + skip) * 64 / kTileKeys;
        if (t >= prefix_tiles && t < from_tile) t = from_tile;
      }
    }
    return min(t, end_tile);
  };

  // ---- masks of the lane's rows
  int row_lo[2], row_span[2];
#pragma unroll
  for (int qc = 0; qc < 2; ++qc) {
    const int i = min(wave_row0 + 16 * qc + col, S - 1);
    row_lo[qc] = low(i);
    row_span[qc] = high(i) - row_lo[qc];
  }
  // Whether the lane's row of block qc sees a key whose document is id (-1: none).
  auto sees = [&](int qc, int key, int id) -> bool {
    const bool near = static_cast<unsigned>(key - row_lo[qc]) <= static_cast<unsigned>(row_span[qc]);
    return ((near) | (key < prefix)) & (id == row_doc[qc]);
  };
  const float row_at = static_cast<float>(wave_row0 + col);
  const float slope = kBiases && a.slopes != nullptr ? a.slopes[head] * opl::kLog2e : 0.0f;

  // ---- copies of a tile: byte offset of the lane's chunks, swizzled
  int k_src[kCopies], v_src[kCopies];
#pragma unroll
  for (int j = 0; j < kCopies; ++j) {
    const int slot = (wave * kCopies + j) * 64 + lane;
    const int row = slot / L::kChunks;
    const int phys = slot % L::kChunks;
    const int kd = L::kElems * (phys ^ L::swizzle_k(row));
    const int vd = L::kElems * (phys ^ L::swizzle_v(row));
    k_src[j] = kd < dm ? (row * static_cast<int>(a.ks.token) + kd) * L::kSize : kNoData;
    v_src[j] = vd < dm ? (row * static_cast<int>(a.vs.token) + vd) * L::kSize : kNoData;
  }
  const unsigned k_bytes = static_cast<unsigned>((S - 1) * a.ks.token + dm) * L::kSize;
  const unsigned v_bytes = static_cast<unsigned>((S - 1) * a.vs.token + dm) * L::kSize;
  const int wave_s = __builtin_amdgcn_readfirstlane(wave);
  // key0 < S: the ranges stay positive. (Ids behind the last read as 0: such keys
  // are outside every row's bounds.)
  auto issue = [&](unsigned char* st, int* ids, int key0) {
    if (docs != nullptr && wave_s == 0)
      opl::buffer_copy4_lds(docs + key0, static_cast<unsigned>(S - key0) * 4, ids, lane * 4);
    const std::size_t k_at = static_cast<std::size_t>(key0) * a.ks.token;
    const std::size_t v_at = static_cast<std::size_t>(key0) * a.vs.token;
    const unsigned k_rest = k_bytes - static_cast<unsigned>(k_at) * L::kSize;
    const unsigned v_rest = v_bytes - static_cast<unsigned>(v_at) * L::kSize;
#pragma unroll
    for (int j = 0; j < kCopies; ++j)
      opl::buffer_copy16_lds(kh + k_at, k_rest, st + (wave_s * kCopies + j) * 1024, k_src[j]);
#pragma unroll
    for (int j = 0; j < kCopies; ++j)
      opl::buffer_copy16_lds(vh + v_at, v_rest, st + L::kTile + (wave_s * kCopies + j) * 1024, v_src[j]);
  };
  int k_off[L::kSteps];
#pragma unroll
  for (int c = 0; c < L::kSteps; ++c)
    k_off[c] = col * L::kRowBytes + (((4 * c + quad) ^ L::swizzle_k(col)) * 16);
  int v_base[L::kDBlocks];
#pragma unroll
  for (int db = 0; db < L::kDBlocks; ++db) {
    if constexpr (kHalf) {
      const int row = 4 * quad + col / 4;
      const int d = 16 * db + 4 * (col % 4);
      v_base[db] = L::kTile + row * L::kRowBytes + (((d >> 3) ^ L::swizzle_v(row)) * 16) + (d & 7) * 2;
    } else {
      const int row = 4 * quad;
      const int d = 16 * db + col;
      v_base[db] = L::kTile + row * L::kRowBytes + (((d >> 2) ^ L::swizzle_v(row)) * 16) + (d & 3) * 4;
    }
  }

  // ---- state: lane l holds query 16 qc + col, dims 16 db + 4 quad + e of O^T
  floatx4 o[2][L::kDBlocks];
  float row_max[2], move_above[2], lane_sum[2], row_sum[2];
  floatx4 sums[2];
  half8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = static_cast<_Float16>(1.0f);
  // The scores' scale in the exponent; where they are biased they get it before.
  const float scale_of_scores = kCaps ? a.rules.template after<kPrecise>() : a.rules.scale;
  const float scale = kBiases ? 1.0f : scale_of_scores;
  const float inv_scale = 1.0f / scale;

  bool exact = false;  // uniform over the workgroup
  for (;;) {
#pragma unroll
    for (int qc = 0; qc < 2; ++qc) {
#pragma unroll
      for (int db = 0; db < L::kDBlocks; ++db) o[qc][db] = floatx4{0, 0, 0, 0};
      sums[qc] = floatx4{0, 0, 0, 0};
      lane_sum[qc] = 0.0f;
      row_max[qc] = -FLT_MAX;
      move_above[qc] = -INFINITY;
    }

    auto body = [&](const unsigned char* cur, const int* ids, int key0, bool whole, bool bounds) {
      constexpr int kHalves = kTileKeys / 32;
      floatx4 s[kHalves][2][2];  // [32 keys][16 keys][qc]
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int j = 0; j < kHalves; ++j) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int qc = 0; qc < 2; ++qc) s[j][kb][qc] = floatx4{0, 0, 0, 0};
        if constexpr (kHalf) {
          half8 f[2][L::kSteps];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int c = 0; c < L::kSteps; ++c)
              f[kb][c] = *reinterpret_cast<const half8*>(cur + k_off[c] + (32 * j + 16 * kb) * L::kRowBytes);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int c = 0; c < L::kSteps; ++c)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int qc = 0; qc < 2; ++qc)
                s[j][kb][qc] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[kb][c], qf[qc][c], s[j][kb][qc], 0, 0, 0);
        } else {
#pragma unroll
          for (int c = 0; c < L::kSteps; ++c) {
            floatx4 f[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
              f[kb] = *reinterpret_cast<const floatx4*>(cur + k_off[c] + (32 * j + 16 * kb) * L::kRowBytes);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int qc = 0; qc < 2; ++qc)
                  s[j][kb][qc] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[kb][e], qf[qc][c][e], s[j][kb][qc], 0, 0, 0);
          }
        }
        // Capped and biased, between the products of the two halves and without a
        // branch: the vector units work on one while the matrix cores compute the
        // other (8000 tokens causal, capped 637 -> 590 us, biased 632 -> 587; a
        // polynomial for tanh instead of v_exp and v_rcp was no faster).
        if constexpr (kRules != kScaled) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int qc = 0; qc < 2; ++qc)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float x = s[j][kb][qc][e];
                if constexpr (kCaps) x = a.rules.template capped<kPrecise>(x);
                if constexpr (kBiases) {  // (positions are below 2^20: exact)
                  const float from = row_at - static_cast<float>(key0 + 4 * quad);
                  x = fmaf(x, scale_of_scores, -slope * fabsf(from + (16 * qc - 32 * j - 16 * kb - e)));
                }
                s[j][kb][qc][e] = x;
              }
        }
      }
      __builtin_amdgcn_s_setprio(0);
      if (bounds) {  // three instructions a score instead of eight (window 320: 88.8 -> 82.0 us)
#pragma unroll
        for (int qc = 0; qc < 2; ++qc) {
          const int from = key0 + 4 * quad - row_lo[qc];
#pragma unroll
          for (int j = 0; j < kHalves; ++j)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                s[j][kb][qc][e] = static_cast<unsigned>(from + 32 * j + 16 * kb + e) <=
                                          static_cast<unsigned>(row_span[qc])
                                      ? s[j][kb][qc][e]
                                      : -INFINITY;
        }
      } else if (!whole) {
#pragma unroll
        for (int j = 0; j < kHalves; ++j)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            const int at = 32 * j + 16 * kb + 4 * quad;
            const int key = key0 + at;
            int4 id = make_int4(0, 0, 0, 0);
            if (docs != nullptr) id = *reinterpret_cast<const int4*>(ids + at);
            const int of[4] = {max(id.x, -1), max(id.y, -1), max(id.z, -1), max(id.w, -1)};
#pragma unroll
            for (int qc = 0; qc < 2; ++qc)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                s[j][kb][qc][e] = sees(qc, key + e, of[e]) ? s[j][kb][qc][e] : -INFINITY;
          }
      }
      float raw[2];
#pragma unroll
      for (int qc = 0; qc < 2; ++qc) raw[qc] = s[0][0][qc][0];
#pragma unroll
      for (int j = 0; j < kHalves; ++j)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int qc = 0; qc < 2; ++qc)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              raw[qc] = __builtin_elementwise_maximum(raw[qc], s[j][kb][qc][e]);
      if (__builtin_amdgcn_ballot_w64(raw[0] > move_above[0] || raw[1] > move_above[1]) != 0) {
#pragma unroll
        for (int qc = 0; qc < 2; ++qc) {
          const float top = opl::max_lane_xor32(opl::combine_xor16_f32<opl::MaxOp>(raw[qc]));
          const float new_max = fmaxf(row_max[qc], top * scale);
          const float alpha = opl::fast_exp2(row_max[qc] - new_max);
          row_max[qc] = new_max;
          move_above[qc] = (new_max + kLazyLog2) * inv_scale;
          if constexpr (kHalf) sums[qc] *= alpha;
          else lane_sum[qc] *= alpha;
#pragma unroll
          for (int db = 0; db < L::kDBlocks; ++db) o[qc][db] *= alpha;
        }
      }
#pragma unroll
      for (int j = 0; j < kHalves; ++j) {
        const int rows = 32 * j * L::kRowBytes;
        if constexpr (kHalf) {
          half8 p[2];
#pragma unroll
          for (int qc = 0; qc < 2; ++qc)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                p[qc][4 * kb + e] = static_cast<_Float16>(opl::fast_exp2(
                    fmaf(s[j][kb][qc][e], scale, -row_max[qc])));
#pragma unroll
          for (int db = 0; db < L::kDBlocks; ++db) {
            const fp16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4f16((OPL_LDS fp16x4*)(cur + v_base[db] + rows));
            const fp16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4f16(
                (OPL_LDS fp16x4*)(cur + v_base[db] + rows + 16 * L::kRowBytes));
            half8 f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              f[e] = lo4[e];
              f[4 + e] = hi4[e];
            }
#pragma unroll
            for (int qc = 0; qc < 2; ++qc)
              o[qc][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, p[qc], o[qc][db], 0, 0, 0);
          }
#pragma unroll
          for (int qc = 0; qc < 2; ++qc)
            sums[qc] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, p[qc], sums[qc], 0, 0, 0);
        } else {
          float p[2][2][4];
#pragma unroll
          for (int qc = 0; qc < 2; ++qc)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                p[qc][kb][e] = opl::fast_exp2(
                    fmaf(s[j][kb][qc][e], scale, -row_max[qc]));
                lane_sum[qc] += p[qc][kb][e];
              }
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float f[L::kDBlocks];
#pragma unroll
              for (int db = 0; db < L::kDBlocks; ++db) {
                f[db] = *reinterpret_cast<const float*>(cur + v_base[db] + rows + (16 * kb + e) * L::kRowBytes);
              }
#pragma unroll
              for (int db = 0; db < L::kDBlocks; ++db)
#pragma unroll
                for (int qc = 0; qc < 2; ++qc)
                  o[qc][db] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[db], p[qc][kb][e], o[qc][db], 0, 0, 0);
            }
        }
      }
    };

    // One tile: `t` is in cur; the copy of the group's next tile goes to nxt.
    auto advance = [&](int t) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) t = visit(t + 1);
      return t;
    };
    struct Marks {
      unsigned within = 1, one = 1;  // (without documents)
    } marks;
    auto read_marks = [&](int t) {
      Marks m;
      const int bit = t * kTileKeys / 64;
      m.one = 0;
      if (bit < kMarkWords * 32) {
        m.within = (some[wave][bit / 32] >> (bit % 32)) & 1;
        m.one = (single[wave][bit / 32] >> (bit % 32)) & 1;
      }
      return m;
    };
    // Exact pass: non-finite values of the arrived tile become zeros.
    auto drop_non_finite = [&](unsigned char* cur) {  // (by the group's wavefronts)
      const int first = (kW == 1 ? 0 : wave) * opl::kWaveSize + lane;
      for (int i = first; i < L::kTile / L::kSize; i += kW * opl::kWaveSize) {
        T* const x = reinterpret_cast<T*>(cur + L::kTile) + i;
        if (!(fabsf(static_cast<float>(*x)) < INFINITY)) *x = T(0);
      }
    };
    auto tile = [&](const unsigned char* cur, const int* ids, unsigned char* nxt, int* ids_nxt, int t) {
      const int after = t < end_tile ? advance(t) : end_tile;
      if (after < end_tile) issue(nxt, ids_nxt, after * kTileKeys);
      const unsigned within = marks.within, one = marks.one;  // of this tile, read a tile ahead
      if (docs != nullptr) marks = read_marks(after);
      __builtin_amdgcn_sched_barrier(0);
      if (exact) {
        if (t < end_tile) drop_non_finite(const_cast<unsigned char*>(cur));
        __builtin_amdgcn_s_waitcnt(0);
        if constexpr (kW > 1) __syncthreads();  // (all groups, also those without a tile)
      }
      const int key0 = t * kTileKeys;
      const int key1 = key0 + kTileKeys - 1;
      const int row0 = wave_row0, row1 = min(wave_row0 + kRowsPerWave, S) - 1;
      if (t < end_tile && row0 < S &&
          (key0 < prefix || (key1 >= low(row0) && key0 <= high(row1)))) {
        bool whole = key1 < prefix || (key0 >= low(row1) && key1 <= high(row0));
        whole = whole && one != 0;
        const bool bounds = !whole && one != 0 && key0 >= prefix;  // alone decide
        if (within != 0) body(cur, ids, key0, whole, bounds);
      }
      __builtin_amdgcn_s_waitcnt(0);
      if constexpr (kW == 1) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      } else {
        __syncthreads();
      }
      return after;
    };
    int t = visit(0);
    for (int g = 0; g < group; ++g) t = visit(t + 1);
    if (t < end_tile) issue(st0, id0, t * kTileKeys);
    if (docs != nullptr) marks = read_marks(t);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if constexpr (kGroups == 1 || kW == 1) {
      while (t < end_tile) {  // uniform over the wavefronts that meet at the barrier
        t = tile(st0, id0, st1, id1, t);
        if (t >= end_tile) break;
        t = tile(st1, id1, st0, id0, t);
      }
    } else {
      // Groups of more wavefronts meet at the workgroup's barrier: all run as
      // many steps as the first group, which has the most tiles.
      int lead = visit(0);
      while (lead < end_tile) {
        lead = advance(lead);
        t = tile(st0, id0, st1, id1, t);
        if (lead >= end_tile) break;
        lead = advance(lead);
        t = tile(st1, id1, st0, id0, t);
      }
    }
    // Every lane of a row has its max and sum; the groups exchange them. A NaN in
    // the sum of a wavefront's O: a non-finite value was multiplied by a hidden
    // key's 0, or is seen (or infinities of both signs are).
    float all[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int qc = 0; qc < 2; ++qc) {
      row_sum[qc] = kHalf ? sums[qc][0]
                          : opl::sum_lane_xor32(opl::combine_xor16_f32<opl::SumOp>(lane_sum[qc]));
      if (kGroups > 1 && quad == 0)
        ends[group * kW + wave][16 * qc + col] = make_float2(row_max[qc], row_sum[qc]);
#pragma unroll
      for (int db = 0; db < L::kDBlocks; ++db)
#pragma unroll
        for (int e = 0; e < 4; ++e) all[e] += o[qc][db][e];
    }
    const float sum = (all[0] + all[1]) + (all[2] + all[3]);
    const bool bad = __builtin_amdgcn_ballot_w64(sum != sum) != 0;
    if (lane == 0) poisoned[threadIdx.x / opl::kWaveSize] = bad && !exact;
    __syncthreads();  // every stage is free
    bool again = false;
#pragma unroll
    for (int i = 0; i < kGroups * kW; ++i) again |= poisoned[i];
    if (!__builtin_amdgcn_readfirstlane(again)) break;
    exact = true;
    __syncthreads();  // (all have read the flags)
  }
  // ---- join the groups, normalise, store whole rows through LDS
  float coef[2];
  auto inverse = [](float l) { return l > 0.0f || l != l ? 1.0f / l : 0.0f; };
#pragma unroll
  for (int qc = 0; qc < 2; ++qc) {
    if constexpr (kGroups > 1) {
      float2 of[kGroups];
      float m = -FLT_MAX, l = 0.0f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        of[g] = ends[g * kW + wave][16 * qc + col];
        m = fmaxf(m, of[g].x);
      }
#pragma unroll
      for (int g = 0; g < kGroups; ++g) l += of[g].y * opl::fast_exp2(of[g].x - m);
      coef[qc] = opl::fast_exp2(row_max[qc] - m) * inverse(l);
    } else {
      coef[qc] = inverse(row_sum[qc]);
    }
  }
#pragma unroll
  for (int qc = 0; qc < 2; ++qc)
#pragma unroll
    for (int db = 0; db < L::kDBlocks; ++db) o[qc][db] *= coef[qc];
  if (exact) {
    // The non-finite values go to the rows that see their keys, after the
    // weights (infinity times a weight of 0 is NaN); one group adds them, as
    // the groups' O are summed.
    typedef T Four __attribute__((ext_vector_type(4)));
    for (int t = group == 0 ? visit(0) : end_tile; t < end_tile; t = visit(t + 1)) {
      for (int key = t * kTileKeys; key < min((t + 1) * kTileKeys, S); ++key) {
        const int id = docs != nullptr ? max(docs[key], -1) : 0;
        const T* const row = vh + static_cast<std::int64_t>(key) * a.vs.token;
#pragma unroll
        for (int db = 0; db < L::kDBlocks; ++db) {
          const int d = 16 * db + 4 * quad;
          const Four x = *reinterpret_cast<const Four*>(row + (d < dm ? d : 0));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float y = static_cast<float>(x[e]);
            if (fabsf(y) < INFINITY) continue;
#pragma unroll
            for (int qc = 0; qc < 2; ++qc) o[qc][db][e] += sees(qc, key, id) ? y : 0.0f;
          }
        }
      }
    }
  }
  // (One group stores what it has: fp16 is rounded before the exchange.)
  typedef typename std::conditional<kGroups == 1, T, float>::type Stage;
  typedef Stage StageFour __attribute__((ext_vector_type(4)));
  constexpr int kBlockBytes = kRowsPerWave * D * static_cast<int>(sizeof(Stage));
  constexpr int kPerArray = kArray / kBlockBytes;
  static_assert(kPerArray >= 1 && kGroups * kW <= 2 * kPerArray, "blocks fit the stage arrays");
  auto block = [&](int index) -> StageFour* {
    return reinterpret_cast<StageFour*>(index < kPerArray ? stage0 + index * kBlockBytes
                                                          : stage1 + (index - kPerArray) * kBlockBytes);
  };
  constexpr int kQuads = D / 4;                        // groups of 4 dims in a row
  constexpr int kQuadsPerLane = L::kElems / 4;         // of a lane's 16-byte store
  auto swizzle = [](int row) { return row * kQuadsPerLane % kQuads; };
  {
    StageFour* const to = block(group * kW + wave);
#pragma unroll
    for (int qc = 0; qc < 2; ++qc)
#pragma unroll
      for (int db = 0; db < L::kDBlocks; ++db) {
        const int r = 16 * qc + col;
        StageFour x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = static_cast<Stage>(o[qc][db][e]);
        to[r * kQuads + ((4 * db + quad) ^ swizzle(r))] = x;
      }
  }
  if constexpr (kGroups > 1) __syncthreads();  // (else a wavefront reads what it wrote)
  // Each wavefront stores 32 / kGroups rows of its block's kGroups copies.
  constexpr int kLanes = D / L::kElems;                // lanes per row
  constexpr int kRowsPerStore = opl::kWaveSize / kLanes;
  constexpr int kWaveRows = kRowsPerWave / kGroups;
  typedef T Out __attribute__((ext_vector_type(L::kElems)));
  const int v = group * kW + wave;
  const int bw = v / kGroups;
  const int cc = lane % kLanes;
  T* const obase = a.out + batch * a.os.batch + head * a.os.head;
#pragma unroll
  for (int i = 0; i < kWaveRows / kRowsPerStore; ++i) {
    const int row = (v % kGroups) * kWaveRows + kRowsPerStore * i + lane / kLanes;
    Out y;
#pragma unroll
    for (int j = 0; j < kQuadsPerLane; ++j) {
      const int at = row * kQuads + ((cc * kQuadsPerLane + j) ^ swizzle(row));
      StageFour x = block(bw)[at];
#pragma unroll
      for (int g = 1; g < kGroups; ++g) x += block(g * kW + bw)[at];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[4 * j + e] = static_cast<T>(x[e]);
    }
    const int token = q0 + kRowsPerWave * bw + row;
    if (token < S && L::kElems * cc < dm)
      *reinterpret_cast<Out*>(obase + token * a.os.token + L::kElems * cc) = y;
  }
}

template <typename T, int D, int Dc, int kGroups, int kW, int kTileKeys>
hipError_t launch(const MaskedArgs<T>& a, hipStream_t stream) {
  constexpr int kRows = kRowsPerWave * kW;
  const long long blocks = (a.S + kRows - 1LL) / kRows * a.bh;
  const dim3 grid(static_cast<unsigned>((blocks + kXcds - 1) / kXcds * kXcds));
  const dim3 block(kGroups * kW * opl::kWaveSize);
  const bool capped = a.rules.cap != 0.0f, biased = a.slopes != nullptr;
  const bool wide_cap = sizeof(T) == 2 && a.rules.wide_cap();
  if (capped && (biased || wide_cap))
    masked_attention_kernel<T, D, Dc, kGroups, kW, kTileKeys, kBoth><<<grid, block, 0, stream>>>(a);
  else if (capped)
    masked_attention_kernel<T, D, Dc, kGroups, kW, kTileKeys, kCapped><<<grid, block, 0, stream>>>(a);
  else if (biased)
    masked_attention_kernel<T, D, Dc, kGroups, kW, kTileKeys, kBiased><<<grid, block, 0, stream>>>(a);
  else
    masked_attention_kernel<T, D, Dc, kGroups, kW, kTileKeys, kScaled><<<grid, block, 0, stream>>>(a);
  return hipGetLastError();
}

// G key groups of W wavefronts, tiles of K keys: head dims up to 64, and past it.
template <typename T, int G, int W, int K>
hipError_t narrow(const MaskedArgs<T>& a, hipStream_t stream) {
  return launch<T, 64, 64, G, W, K>(a, stream);
}
template <typename T, int G, int W, int K>
hipError_t wide(const MaskedArgs<T>& a, hipStream_t stream) {
  // Head dims of 65 to 96 compute on 96: fp16 B2 H16 S2999 prefix 106 -> 98 us.
  if (a.dm <= 96) return launch<T, 128, 96, G, W, K>(a, stream);
  return launch<T, 128, 128, G, W, K>(a, stream);
}

// Blocks of 32 to 128 query rows, and keys split between groups of wavefronts
// where the grid of 128-row blocks does not fill the CUs' two workgroups each
// (as attention.hip does). Measured on MI355X (us; groups, wavefronts per group,
// tile keys), B1 unless said, "c" causal:
//   fp16 D64    1,4,64  2,2,64  2,4,64  4,1,32     fp16 D128   1,4,64  2,2,32  2,4,64  4,2,32  4,1,32
//   H12 S131 c    8.2     7.4     8.3     6.4      H12 S131 c   10.8     8.8    10.5     9.0     8.8
//   H32 S500 c   13.9    10.7    12.5     8.9      H12 S500     17.2    14.4    16.2    13.2    12.6
//   H2 S8000    109.9    68.7    86.0    53.8      H32 S500     18.0    15.1    16.7    14.1    23.3
//   H32 S1000    20.1    17.9    18.1    23.9      H4 S4000     82.6    65.1    67.6    52.7    76.2
//   H16 S2000 c  34.0    24.0    27.9    24.6      H32 S1000 c  29.6    24.0    25.7    26.5    45.5
//   B4 H32 S131   8.8    10.0     9.6    12.3      H16 S2000 c  48.4    38.5    40.7    36.8    60.6
//   H32 S2000 c  37.0    34.1    34.3    45.2      H16 S2000    48.0    44.8    40.9    55.7    88.7
//   H32 S2000    44.6    52.8    53.4    66.8      H12 S4000 c  96.3   105.8    80.3   109.8   165.9
//   B4 H32 S500c 16.1    19.7    19.9    27.9      H32 S2000 c  55.2    51.9    49.9    71.7   120.4
//   B2 H32 S1000c 23.4   25.2    24.9    34.5      B2 H32 S1000c 34.7   36.1    36.1    51.8    90.1
// Many heads of up to 192 tokens, whose second 128-row block is nearly empty:
// 1,2,32 (B16 H32 S131 D128 23.7 against 27.3, D64 16.5 against 18.1).
//   fp32 D64    1,4,32  2,2,32  4,1,32  1,2,32     fp32 D128   1,4,32  2,2,32  1,2,32
//   H12 S500 c   43.0    26.1    18.1    41.8      H12 S131 c   26.3    20.8    27.9
//   H8 S2000 c  148.9    85.3    56.2   147.7      H2 S8000     1047     607    1104
//   H8 S2000    149.6    87.6    93.6   149.1      H32 S1000 c 142.5    97.6   149.8
//   H16 S2000   154.4   142.1   181.9   248.8      H32 S1000   145.8   167.0   151.5
//   H32 S2000 c 203.0   164.8   216.1   202.5      H32 S2000 c 361.7   351.0   314.5
//   H12 S4000 window 512 (384 blocks)              B4 H32 S500 c 102.5 117.0    97.7
//               156.7   141.3           139.9      H32 S2000   495.9   632.7   568.1
template <typename T>
hipError_t choose(const MaskedArgs<T>& a, hipStream_t stream) {
  const long long blocks = (a.S + 127LL) / 128 * a.bh;
  const long long blocks32 = (a.S + 31LL) / 32 * a.bh;
  // Keys that a block walks, by the window.
  const long long reach = a.window > 0 ? (a.causal ? 1LL : 2LL) * a.window + 128 : a.S;
  const long long walk = reach < a.S ? reach : a.S;
  if (a.dm > 64) {
    if constexpr (sizeof(T) == 2) {
      if (blocks32 <= 256) return wide<T, 4, 1, 32>(a, stream);
      if (a.S <= 192 && blocks > 256) return wide<T, 1, 2, 32>(a, stream);
      if (blocks <= 128) return wide<T, 4, 2, 32>(a, stream);
      if (a.causal && blocks <= 256 && walk > 192) return wide<T, 2, 2, 32>(a, stream);
      if ((blocks <= 256 && walk > 192) || (a.causal && blocks <= 512 && walk >= 1536))
        return wide<T, 2, 4, 64>(a, stream);
      return wide<T, 1, 4, 64>(a, stream);
    } else {
      if (blocks <= 128 || (a.causal && blocks <= 256 && walk > 192))
        return wide<T, 2, 2, 32>(a, stream);
      if (a.causal && blocks > 256 && blocks <= 512) return wide<T, 1, 2, 32>(a, stream);
      return wide<T, 1, 4, 32>(a, stream);
    }
  }
  if constexpr (sizeof(T) == 2) {
    if (blocks32 <= 512) return narrow<T, 4, 1, 32>(a, stream);
    if (a.S <= 192 && blocks > 256) return narrow<T, 1, 2, 32>(a, stream);
    if (blocks <= 256 && walk > 192) return narrow<T, 2, 2, 64>(a, stream);
    if (a.causal && blocks <= 512 && walk >= 1536) return narrow<T, 2, 4, 64>(a, stream);
    return narrow<T, 1, 4, 64>(a, stream);
  } else {
    if (blocks32 <= (a.causal ? 512 : 256)) return narrow<T, 4, 1, 32>(a, stream);
    if (walk > 192 && (blocks <= 256 || (a.causal && blocks <= 512)))
      return narrow<T, 2, 2, 32>(a, stream);
    if (blocks > 256 && blocks < 512) return narrow<T, 1, 2, 32>(a, stream);
    return narrow<T, 1, 4, 32>(a, stream);
  }
}

template <typename T>
int masked_entry(MaskedArgs<T> a, int batch, int kv_heads, float scale, float softcap,
                 void* stream_handle) {
  const opl::MaskedShape shape = {batch, a.q_heads, kv_heads, a.S, a.dm};
  if (a.q == nullptr || a.k == nullptr || a.v == nullptr || a.out == nullptr ||
      !opl::masked_shape_ok(shape, sizeof(T)) || !opl::score_rules_ok(scale, a.window, softcap) ||
      !opl::masked_strides_ok(a.q, a.qs, shape, sizeof(T)) ||
      !opl::masked_strides_ok(a.k, a.ks, shape, sizeof(T)) ||
      !opl::masked_strides_ok(a.v, a.vs, shape, sizeof(T)) ||
      !opl::masked_strides_ok(a.out, a.os, shape, sizeof(T)))
    return hipErrorInvalidValue;
  a.bh = batch * a.q_heads;
  a.group = a.q_heads / kv_heads;
  a.rules = opl::ScoreRules::of(scale, softcap);
  const hipStream_t stream = static_cast<hipStream_t>(stream_handle);
  return choose(a, stream);
}

opl::MaskedStrides of(operatorlib_strides_t s) { return {s.batch, s.head, s.token}; }

}  // namespace

extern "C" int operatorlib_masked_attention_f16(
    const operatorlib_half_t* q, operatorlib_strides_t q_strides, const operatorlib_half_t* k,
    operatorlib_strides_t k_strides, const operatorlib_half_t* v, operatorlib_strides_t v_strides,
    const float* slopes, const int32_t* documents, const int32_t* prefixes,
    operatorlib_half_t* output, operatorlib_strides_t output_strides, int batch, int q_heads,
    int kv_heads, int sequence, int head_dim, float scale, int causal, int window, float softcap,
    void* stream) {
  const auto in = [](const operatorlib_half_t* p) { return reinterpret_cast<const _Float16*>(p); };
  return masked_entry<_Float16>(
      {in(q), in(k), in(v), reinterpret_cast<_Float16*>(output), of(q_strides), of(k_strides),
       of(v_strides), of(output_strides), slopes, documents, prefixes, 0, q_heads, 1, sequence,
       head_dim, causal != 0, window, {}},
      batch, kv_heads, scale, softcap, stream);
}

extern "C" int operatorlib_masked_attention_f32(
    const float* q, operatorlib_strides_t q_strides, const float* k,
    operatorlib_strides_t k_strides, const float* v, operatorlib_strides_t v_strides,
    const float* slopes, const int32_t* documents, const int32_t* prefixes, float* output,
    operatorlib_strides_t output_strides, int batch, int q_heads, int kv_heads, int sequence,
    int head_dim, float scale, int causal, int window, float softcap, void* stream) {
  return masked_entry<float>({q, k, v, output, of(q_strides), of(k_strides), of(v_strides),
                              of(output_strides), slopes, documents, prefixes, 0, q_heads, 1,
                              sequence, head_dim, causal != 0, window, {}},
                             batch, kv_heads, scale, softcap, stream);
}
