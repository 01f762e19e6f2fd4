#pragma once
// LDS layout of the K and V tiles of the attention kernels that copy them
// global -> LDS directly (attention.hip, masked_attention.hip).

#include <hip/hip_runtime.h>

namespace opl {

// K/V tile layout in LDS for element type T (rows keep their global
// layout, D elements each).
// Dc: the dims computed with (D, or 96 in rows of 128).
template <typename T, int D, int kTileKeys, int Dc = D>
struct Layout {
  static constexpr int kSize = static_cast<int>(sizeof(T));
  static constexpr int kElems = 16 / kSize;  // elements per 16-byte chunk
  static constexpr int kRowBytes = D * kSize;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTile = kTileKeys * kRowBytes;  // one K or V tile
  static constexpr int kStage = 2 * kTile;
  // QK^T fragment steps over d: one 16-byte chunk per lane group covers 32
  // fp16 dims (one MFMA 16x16x32) or 16 fp32 dims (four MFMA 16x16x4).
  static constexpr int kSubK = 4 * kElems;
  static constexpr int kSteps = Dc / kSubK;
  static constexpr int kDBlocks = Dc / 16;  // 16-dim blocks of O^T
  // K rows: 16 consecutive rows read one logical chunk (one 16-lane group)
  // and land on 16 different physical chunks.
  __device__ static int swizzle_k(int row) {
    return kChunks >= 16 ? (row & 15) : ((row >> 1) & 7);
  }
  // V rows, fp16: a ds_read_b64_tr_b16 group reads 8 bytes from each of 4
  // rows (4 lanes per row); the 4 rows, and the next group's 4, land on
  // different banks. fp32: each 16-lane group of a ds_read_b32 reads 64
  // bytes of one row, the four groups rows 4 apart, which land on four
  // different 64-byte bank ranges.
  __device__ static int swizzle_v(int row) {
    if constexpr (kSize == 2)
      return D == 128 ? ((4 * (row & 3)) ^ (2 * ((row >> 2) & 1))) : 2 * ((row >> 1) & 3);
    else
      return 4 * ((row >> 2) & 3);
  }
};

}  // namespace opl
