// Register fragments of the fp32-math kernels (v_mfma_f32_16x16x4_f32): tiles
// of 16 rows streamed from global memory, fp32 or bf16 upcast on load.
//
// Operand layouts (lane l: c = l % 16, g = l / 16; MFMA k-slot = g):
//   row fragment r[j]    = X[c][16 j + 4 g .. + 3]: A or B operand whose k
//                          index is the head dim, element t used by MFMA (j, t);
//   column fragment x[i][db] = X[4 g + i][NJ c + db]: A operand X^T whose k
//                          index is the tile row 4 g + i, M index c = dim NJ c + db;
//   score element i      = S[tile row 4 g + i][stationary row c], which is the
//                          B operand of the product with the column fragments;
//   accumulator acc[db][i] = element (dim NJ (4 g + i) + db) of stationary row c.
// (NJ = DP / 16; DP is head_dim rounded up to 16, 32, 64, 96, 128 or 256; dims
// past head_dim are zeros.)
#pragma once

#include "common.h"

namespace lc {

__device__ __forceinline__ f32x4 mfma16x16x4(float a, float b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// W consecutive elements (W = 1, 2 or 4; p aligned to them) as fp32, in one
// load; the other elements of the result are zeros.
template <typename T, int W>
__device__ __forceinline__ f32x4 load_vec(const T* p) {
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
  if constexpr (W == 1) {
    r[0] = load_f32(p);
  } else if constexpr (sizeof(T) == 4) {
    typedef float vt __attribute__((ext_vector_type(W)));
    const vt x = *reinterpret_cast<const vt*>(p);
#pragma unroll
    for (int e = 0; e < W; ++e) r[e] = x[e];
  } else {
    uint2 u = {0u, 0u};
    if constexpr (W == 2) u.x = *reinterpret_cast<const uint32_t*>(p);
    else u = *reinterpret_cast<const uint2*>(p);
    r = f32x4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u),
              __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u)};
  }
  return r;
}

// The same of dims d0 .. d0 + W - 1 of a row whose dims at or past D are zeros
// and are not read; in single elements unless vec (which implies D % 4 == 0).
template <typename T, int W>
__device__ __forceinline__ f32x4 load_w(const T* row, int d0, int D, bool vec) {
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
  if (vec) {
    if (d0 < D) r = load_vec<T, W>(row + d0);
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e)
      if (d0 + e < D) r[e] = load_f32(row + d0 + e);
  }
  return r;
}

// Row fragments of the 16 rows from row0 (rows at or past nrows are zeros).
template <typename T, int NJ>
__device__ __forceinline__ void load_rows(f32x4 (&r)[NJ], const T* base, int64_t stride, int row0,
                                          int nrows, int D, bool vec, int c, int g) {
  const int row = row0 + c;
  if (vec && D == 16 * NJ && row0 + 16 <= nrows) {  // uniform: a whole tile, no checks per load
    const T* p = base + (int64_t)row * stride + 4 * g;
#pragma unroll
    for (int j = 0; j < NJ; ++j) r[j] = load_vec<T, 4>(p + 16 * j);
  } else {
    const bool ok = row < nrows;
    const T* p = base + (int64_t)(ok ? row : 0) * stride;
#pragma unroll
    for (int j = 0; j < NJ; ++j) r[j] = load_w<T, 4>(p, ok ? 16 * j + 4 * g : D, D, vec);
  }
}

// Column fragments of the 16 rows from row0 (rows at or past nrows are zeros).
template <typename T, int NJ>
__device__ __forceinline__ void load_cols(float (&x)[4][NJ], const T* base, int64_t stride,
                                          int row0, int nrows, int D, bool vec, int c, int g) {
  constexpr int W = NJ % 4 == 0 ? 4 : (NJ % 2 == 0 ? 2 : 1);
  const bool whole = vec && D == 16 * NJ && row0 + 16 <= nrows;
  if (whole) {
    const T* p = base + (int64_t)(row0 + 4 * g) * stride + NJ * c;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < NJ / W; ++e) {
        const f32x4 r = load_vec<T, W>(p + i * stride + W * e);
#pragma unroll
        for (int k = 0; k < W; ++k) x[i][W * e + k] = r[k];
      }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + 4 * g + i;
      const bool ok = row < nrows;
      const T* p = base + (int64_t)(ok ? row : 0) * stride;
#pragma unroll
      for (int e = 0; e < NJ / W; ++e) {
        const f32x4 r = load_w<T, W>(p, ok ? NJ * c + W * e : D, D, vec);
#pragma unroll
        for (int k = 0; k < W; ++k) x[i][W * e + k] = r[k];
      }
    }
  }
}

// Keeps the loads of a phase from moving into an earlier one: each operand's
// registers are reloaded one phase after their last use, which is as far
// ahead as the register file allows at head_dim 128.
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

// S (or dP) of one 16 x 16 tile: rows of a against the stationary rows b.
// Two accumulators halve the dependent chain; PARTS restarts keep the sums as
// short as four-lane dot products have them (two: the output of 1,000 causal
// tokens, 32/8 heads of 128, is 2.8e-7 from float64, with one 3.1e-7).
template <int NJ, int PARTS, typename Frag>
__device__ __forceinline__ f32x4 score_tile(const f32x4 (&a)[NJ], const Frag& b) {
  constexpr int kPer = NJ >= PARTS ? NJ / PARTS : NJ;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j0 = 0; j0 < NJ; j0 += kPer) {
    f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
    for (int j = j0; j < j0 + kPer; ++j) {
      const f32x4 bj = b[j];
      s0 = mfma16x16x4(a[j][0], bj[0], s0);
      s1 = mfma16x16x4(a[j][1], bj[1], s1);
      s0 = mfma16x16x4(a[j][2], bj[2], s0);
      s1 = mfma16x16x4(a[j][3], bj[3], s1);
    }
    sum = j0 == 0 ? s0 + s1 : sum + (s0 + s1);
    if (j0 + kPer < NJ) phase();  // one part's registers at a time
  }
  return sum;
}

// Stationary row fragments: in registers, or (kLds) in LDS, one copy for the
// workgroup, each lane at its own 16 bytes of fragment j.
template <int NJ, bool kLds>
struct RowFrags {
  f32x4 r[NJ];
  __device__ __forceinline__ const f32x4& operator[](int j) const { return r[j]; }
};
template <int NJ>
struct RowFrags<NJ, true> {
  const f32x4* p;  // fragment j of lane l at p[64 j] (p already at the lane)
  __device__ __forceinline__ f32x4 operator[](int j) const { return p[64 * j]; }
};

template <int NJ>
__device__ __forceinline__ void accumulate_tile(f32x4 (&acc)[NJ], const float (&x)[4][NJ],
                                                const f32x4& p) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int db = 0; db < NJ; ++db) acc[db] = mfma16x16x4(x[i][db], p[i], acc[db]);
}

// Row pitch (floats) of a wave's partial accumulators in LDS: 16 rows of DP.
__host__ __device__ constexpr int part_pitch(int dp) { return dp + 4; }

template <int NJ>
__device__ __forceinline__ void store_part(float* part, const f32x4 (&acc)[NJ], int c, int g) {
  float* row = part + c * part_pitch(16 * NJ) + 4 * NJ * g;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int db = 0; db < NJ; ++db) row[NJ * i + db] = acc[db][i];
}

}  // namespace lc
