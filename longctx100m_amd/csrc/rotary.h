// Rotary positions: the angles, and the rotation of rows of heads.
//
// Pair i of a head at position p turns by p f_i, f_i its frequency.  At far
// positions that is many turns (10^8 positions at f = 1: 1.6 10^7), of which fp32
// would leave nothing of the fraction that counts.  So a frequency is kept as a
// 64-bit fraction of a turn, f / 2 pi in units of 2^-64: the product with the
// position, taken modulo 2^64, is the fraction of a turn itself, off by |p| 2^-65
// turns at most (2^-38 at 10^8).
//
// cos and sin are their Taylor series about the nearest quarter turn, |x| <= pi/4:
// the first terms left out are x^12 / 12! < 1.2e-10 and x^11 / 11! < 1.8e-9,
// below the rounding of the result.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace lc {

// The rotation as kernels take it.
struct Turns {
  const uint64_t* turns;  // [half], 2^-64 turns a position; null: no rotation
  int half;               // pairs of a head
  int interleaved;        // pairs (2i, 2i + 1), else (i, i + half)
  float factor;           // of cos and sin
};

// (factor cos, factor sin) of an angle in 2^-64 turns.
__device__ __forceinline__ float2 turn_cos_sin(uint64_t phase, float factor) {
  const uint32_t quarter = ((uint32_t)(phase >> 32) + 0x20000000u) >> 30;
  const int64_t rest = (int64_t)(phase - ((uint64_t)quarter << 62));  // within 2^61
  const float x = (float)(int32_t)(rest >> 30) * 3.6572952e-10f;      // 2 pi 2^-34
  const float y = x * x;
  float c = fmaf(y, -2.7557319e-7f, 2.4801587e-5f);  // -1/10!, 1/8!
  c = fmaf(y, c, -1.3888889e-3f);                    // -1/6!
  c = fmaf(y, c, 4.1666667e-2f);                     // 1/4!
  c = fmaf(y, c, -0.5f);
  c = fmaf(y, c, 1.f);
  float s = fmaf(y, 2.7557319e-6f, -1.9841270e-4f);  // 1/9!, -1/7!
  s = fmaf(y, s, 8.3333333e-3f);                     // 1/5!
  s = fmaf(y, s, -1.6666667e-1f);                    // -1/3!
  s = fmaf(x * y, s, x);
  const float u = quarter & 1 ? s : c, v = quarter & 1 ? c : s;
  return make_float2((quarter + 1) & 2 ? -u * factor : u * factor, quarter & 2 ? -v * factor : v * factor);
}

// N consecutive elements as fp32, by 16-byte accesses (kVec; four bf16: 8-byte
// ones) or one by one.
template <bool kVec, int N>
__device__ __forceinline__ void load_n(float (&x)[N], const float* p) {
  if constexpr (kVec) {
    static_assert(N % 4 == 0, "whole vectors");
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const f32x4 a = reinterpret_cast<const f32x4*>(p)[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = a[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = p[e];
  }
}
template <bool kVec, int N>
__device__ __forceinline__ void load_n(float (&x)[N], const uint16_t* p) {
  if constexpr (kVec) {
    static_assert(N == 8 || N == 4, "one vector");
    typedef uint32_t words __attribute__((ext_vector_type(N / 2)));
    const words w = *reinterpret_cast<const words*>(p);
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      x[2 * e] = __uint_as_float(w[e] << 16);
      x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = bf16_to_f32(p[e]);
  }
}
template <bool kVec, int N>
__device__ __forceinline__ void store_n(float* p, const float (&x)[N]) {
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      reinterpret_cast<f32x4*>(p)[i] = f32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) p[e] = x[e];
  }
}
template <bool kVec, int N>
__device__ __forceinline__ void store_n(uint16_t* p, const float (&x)[N]) {
  if constexpr (kVec) {
    typedef uint32_t words __attribute__((ext_vector_type(N / 2)));
    words w;
#pragma unroll
    for (int e = 0; e < N / 2; ++e)
      w[e] = (uint32_t)f32_to_bf16(x[2 * e]) | ((uint32_t)f32_to_bf16(x[2 * e + 1]) << 16);
    *reinterpret_cast<words*>(p) = w;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) p[e] = f32_to_bf16(x[e]);
  }
}

// Turns N pairs.  Half layout: a holds the first elements, b the second ones;
// interleaved: a and b are 2 N consecutive elements.  cs: (cos, sin) of the pairs.
template <int N>
__device__ __forceinline__ void turn_n(float (&a)[N], float (&b)[N], const float2* cs, int interleaved) {
  if (N > 1 && interleaved) {
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      const float2 p = cs[e], q = cs[N / 2 + e];
      const float x = a[2 * e], y = a[2 * e + 1], z = b[2 * e], w = b[2 * e + 1];
      a[2 * e] = x * p.x - y * p.y;
      a[2 * e + 1] = y * p.x + x * p.y;
      b[2 * e] = z * q.x - w * q.y;
      b[2 * e + 1] = w * q.x + z * q.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float2 p = cs[e];
      const float x = a[e], y = b[e];
      a[e] = x * p.x - y * p.y;
      b[e] = y * p.x + x * p.y;
    }
  }
}

// Rows of heads, by element strides.
struct HeadRows {
  int64_t seq, token, head;
};

// The rotation of tokens of several sequences: a workgroup of 256 takes up to
// kTurnTokens of them with all their heads.
constexpr int kTurnTokens = 4;
constexpr int kTurnPairs = 128;  // at most in a head

// Units of N pairs (2 N elements) of `tokens` rows, token t of the workgroup at
// x(t) / out(t) and position pos(t), or absent (there(t) false); dims past the pairs
// are copied, where copy says so.  Requires half % N == 0, and D % 2 N == 0 unless N
// is one.
template <typename T, int N, bool kVec, typename In, typename Out, typename Pos, typename There>
__device__ __forceinline__ void turn_tokens(float2* cs, const Turns& r, int tokens, int heads, int D,
                                            int64_t in_head, int64_t out_head, bool copy,
                                            uint64_t sign, const In& in, const Out& out,
                                            const Pos& pos, const There& there) {
  const int tid = threadIdx.x;
  const int units = ((copy ? D : 2 * r.half) + 2 * N - 1) / (2 * N);  // of a head
  const int step = 256 / units;                    // heads that the workgroup takes at once
  const int u = tid % units, h0 = tid / units;
  const bool turned = N * u < r.half;
  // Where the unit's two groups of N begin.
  const int da = turned && !r.interleaved ? N * u : 2 * N * u;
  const int db = turned && !r.interleaved ? N * u + r.half : 2 * N * u + N;
  const bool both = N > 1 || db < D;  // (a head of odd size ends in half a unit)
  const int rows = tokens * heads;
  const bool mine = h0 < step;
  float a[N], b[N], an[N], bn[N];
  auto load = [&](int t, int h, float (&x)[N], float (&y)[N]) {
    if (!there(t)) return;
    const T* p = in(t) + h * in_head;
    load_n<kVec>(x, p + da);
    if (both) load_n<kVec>(y, p + db);
  };
  int t = h0 / heads, h = h0 - t * heads;
  if (mine && h0 < rows) load(t, h, a, b);  // on its way while the angles are formed
  for (int i = tid; i < tokens * r.half; i += 256) {
    const int at = i / r.half, pair = i - at * r.half;
    cs[i] = turn_cos_sin(sign * (uint64_t)pos(at) * r.turns[pair], r.factor);
  }
  __syncthreads();
  if (!mine) return;
  for (int row = h0; row < rows; row += step) {
    int hn = h + step, tn = t;
    while (hn >= heads) hn -= heads, ++tn;
    if (row + step < rows) load(tn, hn, an, bn);
    if (there(t)) {
      if (turned) turn_n(a, b, cs + t * r.half + N * u, r.interleaved);
      T* p = out(t) + h * out_head;
      store_n<kVec>(p + da, a);
      if (both) store_n<kVec>(p + db, b);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) a[e] = an[e], b[e] = bn[e];
    t = tn;
    h = hn;
  }
}

struct RotaryProblem {
  int dtype;  // 0 = f32, 1 = bf16
  int64_t batch, tokens;
  int heads, D;
  Turns turns;
  bool inverse;
  const int64_t* positions;  // [batch, tokens]; null: pos0 + token
  int64_t pos0;
  const void* x;
  void* out;
  HeadRows xs, os;
  int align;  // of every row, in bytes: 16, 8, or an element's
  bool copy;  // dims that do not turn have to be copied
};
hipError_t launch_rotary(const RotaryProblem& p, hipStream_t s);

}  // namespace lc
