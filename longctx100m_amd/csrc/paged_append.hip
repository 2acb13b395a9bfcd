// New tokens' K and V into a paged cache in e4m3 (gfx950): K turned to its
// position on the way, the tokens' queries turned beside.
//
// A page holds `rows` tokens; a page and KV head has one scale for K and one for
// V, the smallest power of two that brings what it was given to 448 at most.  A
// workgroup takes one page, head and K or V: it reads the new rows of that page
// (K: turns them), reduces their largest magnitude, raises the page's scale if
// it has to, and writes the codes; only if the scale went up does it touch the
// codes of earlier rows.  Rows behind the new ones stay as they are.  So a row
// is read once, and a decoded token costs a row's bytes.  8,192 tokens of 32/8 heads
// of 128 in bf16, queries included, move 185 MB in 43 to 45 us, kernel and call alike (4.1 to
// 4.3 TB/s; 34.5 where one set of inputs again and again stays in the 256 MB cache): the
// pages' workgroups load, reduce over their barrier and store, one phase after the
// other, and the angles are 6 us of instructions.  (Several heads a workgroup, which
// share the angles, need 40 registers more: 58 us.)
//
// Keys are [row][dim] in a page, values [dim][row]: the attention's second
// product wants 16 consecutive keys of one dim in a lane, and gets them with
// plain 16-byte loads.  A thread therefore takes 16 dims of one row of K, and 4
// rows by 8 dims of V, so that it can write a dim's four codes as one word.
#include "e4m3.h"
#include "paged.h"
#include "tile32.h"

#include <algorithm>
#include <type_traits>

namespace lc {
namespace {

struct AppendArgs {
  PagedProblem p;
  Turns turns;
  const void *q, *k, *v;
  void* q_out;
  HeadRows qs, ks, vs;
  int shift;       // log2 of the page's rows
  int touched;     // pages that a sequence's new tokens may lie in
  int kv_blocks;   // workgroups of K and V
  int group;       // tokens of a workgroup of queries
};

// Four fp32 to four e4m3 codes, to nearest even; what is not finite becomes NaN.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
// A word of codes times a power of two <= 1.
__device__ __forceinline__ uint32_t scaled4(uint32_t w, float ratio) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return codes4(lo[0] * ratio, lo[1] * ratio, hi[0] * ratio, hi[1] * ratio);
}
__device__ __forceinline__ float finite_or_nan(float x) { return fabsf(x) < INFINITY ? x : NAN; }
__device__ __forceinline__ float finite_abs(float x) {
  const float y = fabsf(x);
  return y < INFINITY ? y : 0.f;  // NaN too
}

// The largest of the workgroup's values, none negative.
__device__ __forceinline__ float group_max(float x, float* buf) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
  x = group4_max(x);
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = x;
  __syncthreads();
  return fmaxf(fmaxf(buf[0], buf[1]), fmaxf(buf[2], buf[3]));
}

// What a workgroup of K or V writes.
struct Block {
  int64_t token0;  // new token in the page's row 0 (negative: an earlier row)
  int lo, hi;      // new rows of the page
  int head, page;  // (a page that is none is looked at after the new rows are on their way)
  __device__ __forceinline__ int64_t unit(const Pool& p) const { return (int64_t)page * p.Hkv + head; }
};

// IT: 16 values a thread at a time, so many times (a page and head has rows * D).
template <typename T, int IT, bool kVec>
__device__ __forceinline__ void append_keys(const AppendArgs& a, const Block& k, const T* src, int64_t pos0,
                                            float* buf) {
  const int D = a.p.pool.D, units = D / 16;
  const int half = a.turns.turns ? a.turns.half : 0;
  const int u = threadIdx.x % units, r0 = threadIdx.x / units, step = 256 / units;
  const bool turned = 8 * u < half;
  const int da = turned && !a.turns.interleaved ? 8 * u : 16 * u;
  const int db = turned && !a.turns.interleaved ? 8 * u + half : 16 * u + 8;
  float x[IT][8], y[IT][8];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int row = k.lo + r0 + i * step;
    if (r0 < step && row < k.hi) {
      const T* p = src + (k.token0 + row) * a.ks.token;
      load_n<kVec>(x[i], p + da);
      load_n<kVec>(y[i], p + db);
    }
  }
  uint64_t turns[8];
  if (turned)
#pragma unroll
    for (int e = 0; e < 8; ++e) turns[e] = a.turns.turns[8 * u + e];
  if (k.page < 0) return;  // the whole workgroup
  uint8_t* dst = a.p.pool.k + ((k.unit(a.p.pool) * D) << a.shift);
  float* scale = a.p.pool.ks + k.unit(a.p.pool);
  const float was = k.lo > 0 ? *scale : __uint_as_float(kScaleMin);
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int row = k.lo + r0 + i * step;
    if (r0 < step && row < k.hi) {
      if (turned) {
        float2 cs[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) cs[e] = turn_cos_sin((uint64_t)(pos0 + row) * turns[e], a.turns.factor);
        turn_n(x[i], y[i], cs, a.turns.interleaved);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fmaxf(finite_abs(x[i][e]), finite_abs(y[i][e])));
    }
  }
  top = group_max(top, buf);
  const float now = fmaxf(was, __uint_as_float(scale_bits(__float_as_uint(top))));
  const float inv = __uint_as_float(inverse_bits(__float_as_uint(now)));
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int row = k.lo + r0 + i * step;
    if (r0 < step && row < k.hi) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[i][e] = finite_or_nan(x[i][e]) * inv;
        y[i][e] = finite_or_nan(y[i][e]) * inv;
      }
      *reinterpret_cast<uint2*>(dst + row * D + da) = make_uint2(codes4(x[i][0], x[i][1], x[i][2], x[i][3]),
                                                                 codes4(x[i][4], x[i][5], x[i][6], x[i][7]));
      *reinterpret_cast<uint2*>(dst + row * D + db) = make_uint2(codes4(y[i][0], y[i][1], y[i][2], y[i][3]),
                                                                 codes4(y[i][4], y[i][5], y[i][6], y[i][7]));
    }
  }
  if (now > was && k.lo > 0) {  // the whole workgroup
    const float ratio = __uint_as_float(ratio_bits(__float_as_uint(was), __float_as_uint(now)));
    for (int i = threadIdx.x; i < k.lo * units; i += 256) {
      uint4* at = reinterpret_cast<uint4*>(dst) + i;
      uint4 w = *at;
      w.x = scaled4(w.x, ratio), w.y = scaled4(w.y, ratio), w.z = scaled4(w.z, ratio), w.w = scaled4(w.w, ratio);
      *at = w;
    }
  }
  if (threadIdx.x == 0) *scale = now;
}

template <typename T, int IT, bool kVec>
__device__ __forceinline__ void append_values(const AppendArgs& a, const Block& k, const T* src, float* buf) {
  const int D = a.p.pool.D;
  // Four rows from 4 rg, eight dims from 8 dg: row groups across the lanes.
  const int g0 = k.lo / 4, groups = (k.hi + 3) / 4 - g0, items = groups * (D / 8);
  float x[IT][4][8];  // [row][dim]
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int it = threadIdx.x + 256 * i;
    if (it < items) {
      const int dg = it / groups, rg = g0 + it - dg * groups;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 4 * rg + r;
        if (row >= k.lo && row < k.hi) load_n<kVec>(x[i][r], src + (k.token0 + row) * a.vs.token + 8 * dg);
        else
#pragma unroll
          for (int e = 0; e < 8; ++e) x[i][r][e] = 0.f;
      }
    }
  }
  if (k.page < 0) return;  // the whole workgroup
  uint8_t* dst = a.p.pool.v + ((k.unit(a.p.pool) * D) << a.shift);
  float* scale = a.p.pool.vs + k.unit(a.p.pool);
  const float was = k.lo > 0 ? *scale : __uint_as_float(kScaleMin);
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int it = threadIdx.x + 256 * i;
    if (it < items)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, finite_abs(x[i][r][e]));
  }
  top = group_max(top, buf);
  const float now = fmaxf(was, __uint_as_float(scale_bits(__float_as_uint(top))));
  const float inv = __uint_as_float(inverse_bits(__float_as_uint(now)));
  const bool raised = now > was && k.lo > 0;  // the whole workgroup
  const float ratio = __uint_as_float(ratio_bits(__float_as_uint(was), __float_as_uint(now)));
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int it = threadIdx.x + 256 * i;
    if (it < items) {
      const int dg = it / groups, rg = g0 + it - dg * groups;
      const int lo = max(k.lo - 4 * rg, 0), hi = min(k.hi - 4 * rg, 4);  // its new rows
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t* at = reinterpret_cast<uint32_t*>(dst + (((int64_t)8 * dg + e) << a.shift) + 4 * rg);
        float c[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) c[r] = finite_or_nan(x[i][r][e]) * inv;
        const uint32_t w = codes4(c[0], c[1], c[2], c[3]);
        if (lo == 0 && hi == 4) {
          *at = w;
        } else {  // a group with rows of others: their codes stay, or go by the ratio
          const uint32_t mask = (hi == 4 ? ~0u : (1u << 8 * hi) - 1u) & ~((1u << 8 * lo) - 1u);
          const uint32_t low = (1u << 8 * lo) - 1u;
          uint32_t old = *at;
          if (raised) old = (scaled4(old, ratio) & low) | (old & ~low);
          *at = (w & mask) | (old & ~mask);
        }
      }
    }
  }
  if (raised && g0 > 0) {
    for (int i = threadIdx.x; i < g0 * D; i += 256) {  // words of the groups before
      const int d = i / g0;
      uint32_t* at = reinterpret_cast<uint32_t*>(dst + ((int64_t)d << a.shift)) + (i - d * g0);
      *at = scaled4(*at, ratio);
    }
  }
  if (threadIdx.x == 0) *scale = now;
}

template <typename T, int IT, bool kVec>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
  __shared__ float2 cs[kTurnTokens * kTurnPairs];
  __shared__ float buf[4];
  // The queries first: their workgroups stream, those of the pages mostly wait and
  // compute, and fill in behind (8,192 tokens of 32/8 heads of 128, compared when the
  // kernel took 48 us: the pages first 52.5, both in turn 57.5).
  const int q_blocks = gridDim.x - a.kv_blocks;
  if ((int)blockIdx.x >= q_blocks) {
    int x = blockIdx.x - q_blocks;
    const int what = x & 1;
    x >>= 1;
    const int h = x % a.p.pool.Hkv;
    x /= a.p.pool.Hkv;
    const int j = x % a.touched, b = x / a.touched;
    const int past = a.p.past[b];
    const int n = new_tokens(a.p.counts, a.p.N, b, past);
    if (n == 0) return;
    const int64_t at = (int64_t)(past >> a.shift) + j;  // the page's place in the table
    const int64_t row0 = at << a.shift;
    Block k;
    k.token0 = row0 - past;
    k.lo = (int)max((int64_t)0, past - row0);
    k.hi = (int)min((int64_t)1 << a.shift, past + (int64_t)n - row0);
    if (k.lo >= k.hi) return;
    k.head = h;
    k.page = page_of(a.p.table + (int64_t)b * a.p.width, a.p.width, a.p.pool.pages, at);
    if (what == 0)
      append_keys<T, IT, kVec>(a, k, static_cast<const T*>(a.k) + b * a.ks.seq + h * a.ks.head, row0, buf);
    else
      append_values<T, (IT + 1) / 2, kVec>(a, k, static_cast<const T*>(a.v) + b * a.vs.seq + h * a.vs.head, buf);
    return;
  }
  const uint32_t row0 = blockIdx.x * (uint32_t)a.group, rows = (uint32_t)a.p.B * a.p.N;  // below 2^25
  const int n = (int)min((uint32_t)a.group, rows - row0);
  turn_tokens<T, 8, kVec>(
      cs, a.turns, n, a.p.Hq, a.p.pool.D, a.qs.head, a.p.pool.D, true, 1,
      [&](int t) {
        const uint32_t row = row0 + t, b = row / (uint32_t)a.p.N;
        return static_cast<const T*>(a.q) + (int64_t)b * a.qs.seq + (int64_t)(row - b * a.p.N) * a.qs.token;
      },
      [&](int t) { return static_cast<T*>(a.q_out) + (int64_t)(row0 + t) * a.p.Hq * a.p.pool.D; },
      [&](int t) {
        const uint32_t row = row0 + t, b = row / (uint32_t)a.p.N;
        return (int64_t)a.p.past[b] + (row - b * a.p.N);
      },
      [&](int t) {
        const uint32_t row = row0 + t, b = row / (uint32_t)a.p.N;
        return (int)(row - b * a.p.N) < new_tokens(a.p.counts, a.p.N, b, a.p.past[b]);
      });
}

}  // namespace

hipError_t launch_paged_append(const AppendProblem& x, hipStream_t s) {
  AppendArgs a;
  a.p = x.p;
  a.turns = x.turns;
  a.q = x.q;
  a.k = x.k;
  a.v = x.v;
  a.q_out = x.q_out;
  a.qs = x.qs;
  a.ks = x.ks;
  a.vs = x.vs;
  a.shift = __builtin_ctz((unsigned)x.p.pool.rows);
  a.touched = (x.p.N + x.p.pool.rows - 2) / x.p.pool.rows + 1;
  a.kv_blocks = x.p.B * a.touched * x.p.pool.Hkv * 2;
  const int64_t rows = (int64_t)x.p.B * x.p.N;
  a.group = rows <= 1024 ? 1 : kTurnTokens;
  const unsigned grid = (unsigned)(a.kv_blocks + (x.q ? (rows + a.group - 1) / a.group : 0));
  const int units = x.p.pool.D / 16, at_once = 256 / units;  // a row of K, and its rows at once
  const int each = std::max((x.p.pool.rows + at_once - 1) / at_once, (x.p.pool.rows * units + 255) / 256);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, s, a); };
  auto by_type = [&](auto t, auto vec) {
    using T = decltype(t);
    constexpr bool kVec = decltype(vec)::value;
    if (each <= 1) launch(paged_append_kernel<T, 1, kVec>);
    else if (each <= 2) launch(paged_append_kernel<T, 2, kVec>);
    else if (each <= 4) launch(paged_append_kernel<T, 4, kVec>);
    else launch(paged_append_kernel<T, 8, kVec>);
  };
  if (x.p.dtype == 1) {
    if (x.vec) by_type(uint16_t{}, std::true_type{});
    else by_type(uint16_t{}, std::false_type{});
  } else {
    if (x.vec) by_type(float{}, std::true_type{});
    else by_type(float{}, std::false_type{});
  }
  return hipGetLastError();
}

}  // namespace lc
