// Tiles of the kernels that stream a KV cache with a few query rows in
// registers: 8 KB of K or V each, V staged in LDS for transposed reads.
#pragma once

#include "common.h"
#include "tile128.h"

namespace lc {

constexpr int kTileBytes = 8192;   // K (or V) bytes per tile

template <int D>
struct DecodeTile {
  static constexpr int TK = kTileBytes / (2 * D);  // keys per tile
  static constexpr int MB = TK / 16;               // 16-key blocks
  static constexpr int KS = D / 32;                // MFMA k-steps over head_dim
  static constexpr int DB = D / 16;                // 16-dim blocks
};

// V tile in LDS.  head_dim 128: tile128.h's layout.  head_dim 64: rows of 128
// bytes, the eight 16-byte chunks of row r stored at chunk ^ swz64(r).  A
// transposed read serves lanes 0-31 and 32-63 in separate cycles, i.e. eight
// consecutive rows x one chunk pair; rows of equal parity share a half of the
// 256 bytes of banks, and swz64 gives the four of them distinct chunk pairs,
// so the reads are free of bank conflicts.
__device__ __forceinline__ int swz64(int r) { return r & 6; }

template <int D>
struct VTile;
template <>
struct VTile<128> {
  t128::RowLoader<DecodeTile<128>::TK, 1> ld;
  __device__ __forceinline__ void init(int64_t stride, int lane) { ld.init(stride, 0, lane); }
  template <bool kNt = true>
  __device__ __forceinline__ void load(const uint16_t* base, int64_t stride, int row0, int nrows,
                                       uint32_t lds, int lane, const void* filler = nullptr) const {
    ld.template load<false, kNt>(base, stride, row0, nrows, lds, 0, lane, filler);
  }
  static __device__ __forceinline__ int tr_off(int col0, int lane) { return t128::tr_off(0, col0, lane); }
};
template <>
struct VTile<64> {
  static constexpr int kInst = kTileBytes / 1024;  // 8 rows per wave instruction
  uint32_t off[kInst];
  __device__ __forceinline__ void init(int64_t stride, int lane) {
#pragma unroll
    for (int i = 0; i < kInst; ++i) {
      const int r = 8 * i + (lane >> 3);
      off[i] = (uint32_t)(r * stride * 2 + 16 * ((lane & 7) ^ swz64(r)));
    }
  }
  // Rows at or past nrows re-read the last row (callers mask them), or 16 bytes
  // at filler.
  template <bool kNt = true>
  __device__ __forceinline__ void load(const uint16_t* base, int64_t stride, int row0, int nrows,
                                       uint32_t lds, int lane, const void* filler = nullptr) const {
    if (row0 + 8 * kInst <= nrows) {
      const uint8_t* tb = reinterpret_cast<const uint8_t*>(base + (int64_t)row0 * stride);
#pragma unroll
      for (int i = 0; i < kInst; ++i) {
        if constexpr (kNt) t128::dma_b128_nt(tb, off[i], lds + 1024 * i);
        else t128::dma_b128(tb, off[i], lds + 1024 * i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kInst; ++i) {
        const int r = 8 * i + (lane >> 3);
        const int row = min(row0 + r, nrows - 1);
        const uint16_t* g = base + (int64_t)row * stride + 8 * ((lane & 7) ^ swz64(r));
        if (filler != nullptr && row0 + r >= nrows) g = static_cast<const uint16_t*>(filler);
        if constexpr (kNt) t128::dma_b128_nt(g, lds + 1024 * i);
        else t128::dma_b128(g, lds + 1024 * i);
      }
    }
  }
  // Lane 4t + q of group g addresses row 4g + t, columns col0 + 4q .. +3.
  static __device__ __forceinline__ int tr_off(int col0, int lane) {
    const int i = lane & 15, r = 4 * (lane >> 4) + (i >> 2), col = col0 + 4 * (i & 3);
    return r * 128 + 16 * ((col >> 3) ^ swz64(r)) + 2 * (col & 7);
  }
};

}  // namespace lc
