// Attention of a tree of drafted tokens over a KV cache (gfx950).
//
// Token i of sequence b sees the past (rows 0 .. past_b - 1 of the cache) and
// rows past_b + a of its own chain of parents, itself included:
//   m = max s,  l = sum exp(s - m),  o = sum exp(s - m) v / l,  s = q k / sqrt(D).
// The past is the same for every token, the rest is a handful of keys that
// differ from token to token, so the two are computed apart:
//   1. a prefix kernel attends all R = N * Hq / Hkv query rows of a KV head to
//      a split of the past, without any mask, and leaves an unnormalised
//      partial (o, m, l) per row and split;
//   2. cache_merge_kernel, a wave per row, follows the row's chain, takes its
//      few keys with fp32 dot products and merges them with the partials.
// No product with a masked probability exists, so what stands in a row that a
// token does not see cannot reach it, whatever it is.
//
// The lengths are known on the device only.  The host fixes the number of
// split slots (and with it the workspace); each workgroup reads the lengths
// and finds its sequence and key range: slots are dealt out in proportion to
// the sequences' tiles, so a batch of unequal lengths loads the chip evenly.
#include "common.h"
#include "cache.h"
#include "kernels.h"
#include "tile32.h"

#include <algorithm>

namespace lc {
namespace {

constexpr int kTile = 64;  // keys by which the past is dealt out

struct AttnArgs {
  const void *q, *k, *v;
  void* out;
  float *m, *l;
  float *po, *pm, *pl;  // partials: [slots][N * Hq] rows of D, and their statistics (log2 units)
  const int32_t *past, *parents;
  int B, N, C, Hq, Hkv, D, group, R;  // R: query rows of a KV head
  int slots, units;                   // units: workgroups of a slot
  int wave_rows;                      // waves of a workgroup with rows of their own
  int64_t seq, row, head;
  float sl2;
};

// Rows of the past and the tiles they take, at least one (so that every
// sequence has a slot).
__device__ __forceinline__ int past_rows(int past, int C) { return max(0, min(past, C)); }
__device__ __forceinline__ int past_tiles(int past, int C) {
  return max(1, (past_rows(past, C) + kTile - 1) / kTile);
}

__device__ __forceinline__ int wave_sum_i(int x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// The slots of the sequences: sequence b has ceil(tiles_b / per) of them, one
// after another, per = ceil(all tiles / (slots - B)); their number is at most
// all tiles / per + B <= slots.
struct Deal {
  int per;   // tiles of a slot
  int b;     // the sequence looked for
  int first; // its first slot
  int count; // its slots
};
// With slot >= 0 the sequence that has it (count = 0: none), otherwise b's.
__device__ __forceinline__ Deal deal_slots(const int32_t* past, int B, int C, int slots, int slot,
                                           int b) {
  const int lane = threadIdx.x & 63;
  Deal d{};
  if (B == 1) {
    const int t = past_tiles(past[0], C);
    d.per = (t + slots - 2) / (slots - 1);
    d.count = (t + d.per - 1) / d.per;
    if (slot >= d.count) d.count = 0;
    return d;
  }
  int total = 0;
  for (int b0 = 0; b0 < B; b0 += 64)
    total += wave_sum_i(b0 + lane < B ? past_tiles(past[b0 + lane], C) : 0);
  d.per = (total + slots - B - 1) / (slots - B);
  int base = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    const int n = b0 + lane < B ? (past_tiles(past[b0 + lane], C) + d.per - 1) / d.per : 0;
    int end = n;  // inclusive scan
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int x = __shfl_up(end, off, 64);
      if (lane >= off) end += x;
    }
    end += base;
    const bool hit = slot >= 0 ? slot < end && slot >= end - n : b0 + lane == b;
    const uint64_t who = __ballot(hit);
    if (who) {
      const int at = __ffsll((unsigned long long)who) - 1;
      d.b = b0 + at;
      d.count = __shfl(n, at, 64);
      d.first = __shfl(end, at, 64) - d.count;
      return d;
    }
    base = __shfl(end, 63, 64);
  }
  return d;  // a slot without a sequence
}

// The key range of a workgroup.
struct Share {
  int b, k0, k1;  // keys k0 .. k1 - 1 of sequence b (none: k0 == k1)
  int rows;       // its whole past
};
__device__ __forceinline__ bool share_of(const AttnArgs& a, int slot, Share& s) {
  const Deal d = deal_slots(a.past, a.B, a.C, a.slots, slot, 0);
  if (d.count == 0) return false;
  s.b = __builtin_amdgcn_readfirstlane(d.b);
  s.rows = past_rows(a.past[s.b], a.C);
  s.k0 = __builtin_amdgcn_readfirstlane((slot - d.first) * d.per * kTile);
  s.k1 = min(s.k0 + d.per * kTile, s.rows);
  if (s.k0 > s.k1) s.k0 = s.k1;
  return true;
}

// ------------------------------------------------- the past, fp32 products --

// Waves of a workgroup: wave_rows blocks of 16 rows, each by 4 / wave_rows
// waves that take the 16-key tiles in turn and meet in LDS.
template <typename T, int NJ>
__global__ __launch_bounds__(256) void cache_prefix32_kernel(AttnArgs a) {
  constexpr int DP = 16 * NJ;
  constexpr int kPart = 16 * part_pitch(DP);
  __shared__ __attribute__((aligned(16))) float smem[4 * kPart];
  __shared__ float msm[4][16], lsm[4][16];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int slot = blockIdx.x / a.units;
  const int unit = blockIdx.x - slot * a.units;
  const int hk = unit % a.Hkv;
  const int rb = unit / a.Hkv;
  Share s;
  if (!share_of(a, slot, s)) return;  // the whole workgroup

  const int wk = 4 / a.wave_rows;
  const int rsub = wave / wk, ksub = wave - rsub * wk;
  const T* kb = static_cast<const T*>(a.k) + s.b * a.seq + hk * a.head;
  const T* vb = static_cast<const T*>(a.v) + s.b * a.seq + hk * a.head;

  const int r = 16 * (rb * a.wave_rows + rsub) + c;
  const bool rok = r < a.R;
  f32x4 qr[NJ], o[NJ];
  {
    const int rr = rok ? r : 0;
    const int64_t qi = ((int64_t)s.b * a.N + rr / a.group) * a.Hq + hk * a.group + rr % a.group;
    const T* qp = static_cast<const T*>(a.q) + qi * a.D;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      qr[j] = load_w<T, 4>(qp, rok ? 16 * j + 4 * g : a.D, a.D, true);
      o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  float m = -INFINITY, l = 0.f;

  f32x4 kr[NJ];
  float vc[4][NJ];
  const int t0 = s.k0 / 16 + ksub, t1 = (s.k1 + 15) / 16;
  if (t0 < t1) {
    load_rows<T, NJ>(kr, kb, a.row, 16 * t0, s.k1, a.D, true, c, g);
    load_cols<T, NJ>(vc, vb, a.row, 16 * t0, s.k1, a.D, true, c, g);
  }
  for (int t = t0; t < t1; t += wk) {
    f32x4 p = score_tile<NJ, 2>(kr, qr);
    phase();
    const bool more = t + wk < t1;
    if (more) load_rows<T, NJ>(kr, kb, a.row, 16 * (t + wk), s.k1, a.D, true, c, g);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = 16 * t + 4 * g + i >= s.k1 ? -INFINITY : p[i] * a.sl2;
      top = fmaxf(top, p[i]);
    }
    const float mnew = fmaxf(m, group4_max(top));
    if (__any(mnew > m)) {
      const float alpha = mnew > m ? exp2f(m - mnew) : 1.f;  // m = -inf: 0
      l *= alpha;
#pragma unroll
      for (int j = 0; j < NJ; ++j) o[j] *= alpha;
      m = mnew;
    }
    const float muse = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = exp2f(p[i] - muse);
    l += (p[0] + p[1]) + (p[2] + p[3]);
    accumulate_tile<NJ>(o, vc, p);
    phase();
    if (more) load_cols<T, NJ>(vc, vb, a.row, 16 * (t + wk), s.k1, a.D, true, c, g);
  }

  // The waves of a row block meet: each brings its partial to their maximum.
  l = group4_sum(l);
  if (g == 0) msm[wave][c] = m;
  __syncthreads();
  float top = -INFINITY;
  for (int w = 0; w < wk; ++w) top = fmaxf(top, msm[rsub * wk + w][c]);
  const float f = m == -INFINITY ? 0.f : exp2f(m - top);
#pragma unroll
  for (int j = 0; j < NJ; ++j) o[j] *= f;
  if (g == 0) lsm[wave][c] = l * f;
  store_part<NJ>(smem + wave * kPart, o, c, g);
  __syncthreads();
  const int per_row = a.D / 4;
  const int64_t prow0 = (int64_t)slot * a.N * a.Hq;
  for (int i = threadIdx.x; i < 16 * a.wave_rows * per_row; i += 256) {
    const int lr = i / per_row, d = 4 * (i - lr * per_row);
    const int row = 16 * rb * a.wave_rows + lr;
    if (row >= a.R) break;
    const int w0 = lr / 16 * wk, cc = lr % 16;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float ls = 0.f, mt = -INFINITY;
    for (int w = w0; w < w0 + wk; ++w) {
      acc += *reinterpret_cast<const f32x4*>(smem + w * kPart + cc * part_pitch(DP) + d);
      ls += lsm[w][cc];
      mt = fmaxf(mt, msm[w][cc]);
    }
    const int64_t pr = prow0 + (int64_t)(row / a.group) * a.Hq + hk * a.group + row % a.group;
    *reinterpret_cast<f32x4*>(a.po + pr * a.D + d) = acc;
    if (d == 0) {
      a.pm[pr] = mt;
      a.pl[pr] = ls;
    }
  }
}

// ------------------------------------------------ own chain and the merge --

__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <typename T>
__device__ __forceinline__ void store_vec4(T* p, const f32x4& r) {
  if constexpr (sizeof(T) == 4) store4(p, nullptr, r);
  else store4(nullptr, p, r);
}

// A wave per query row.  Lane 16 u + j holds 4-element chunks j, j + 16, .. of
// the head dim for the u-th of every four keys (splits).  NI: such chunks.
template <typename T, int NI>
__global__ __launch_bounds__(256) void cache_merge_kernel(AttnArgs a) {
  __shared__ uint16_t chain_s[4][kCacheMaxTokens];
  __shared__ float score_s[4][kCacheMaxTokens];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = lane & 15, u = lane >> 4;
  const int nrows = a.B * a.N * a.Hq;
  const int row = blockIdx.x * 4 + wave;
  if (row >= nrows) return;  // waves work by themselves: no barrier follows
  const int h = row % a.Hq;
  const int bi = row / a.Hq;
  const int i = bi % a.N, b = bi / a.N;
  const int hk = h / a.group;
  const int past = __builtin_amdgcn_readfirstlane(a.past[b]);

  // The chain of parents, the token itself first.
  uint16_t* chain = chain_s[wave];
  float* score = score_s[wave];
  bool there = past >= 0 && past < a.C && i < a.C - past;
  int n = 0;
  if (there) {
    int par[kCacheMaxTokens / 64];
#pragma unroll
    for (int x = 0; x < kCacheMaxTokens / 64; ++x) {
      const int at = 64 * x + lane;
      par[x] = at < a.N ? (a.parents ? a.parents[(int64_t)b * a.N + at] : at - 1) : -2;
    }
    int at = i;
    while (true) {  // at falls with every step
      if (lane == 0) chain[n] = (uint16_t)at;
      ++n;
      int p = -2;
#pragma unroll
      for (int x = 0; x < kCacheMaxTokens / 64; ++x)
        if (at >> 6 == x) p = __builtin_amdgcn_readlane(par[x], at & 63);
      if (p == -1) break;
      if (p < -1 || p >= at) {
        there = false;
        break;
      }
      at = p;
    }
  }
  const int64_t si = ((int64_t)b * a.Hq + h) * a.N + i;
  T* out = static_cast<T*>(a.out) + (int64_t)row * a.D;
  const int nch = a.D / 4;
  if (!there) {
#pragma unroll
    for (int x = 0; x < NI; ++x)
      if (u == 0 && j + 16 * x < nch) store_vec4<T>(out + 4 * (j + 16 * x), f32x4{0.f, 0.f, 0.f, 0.f});
    if (lane == 0) {
      if (a.m) a.m[si] = -INFINITY;
      if (a.l) a.l[si] = 0.f;
    }
    return;
  }
  wave_lds_sync();

  f32x4 qv[NI];
  const T* qp = static_cast<const T*>(a.q) + (int64_t)row * a.D;
#pragma unroll
  for (int x = 0; x < NI; ++x) qv[x] = load_w<T, 4>(qp, 4 * (j + 16 * x), a.D, true);
  const T* kb = static_cast<const T*>(a.k) + b * a.seq + hk * a.head + past * a.row;
  const T* vb = static_cast<const T*>(a.v) + b * a.seq + hk * a.head + past * a.row;
  float top = -INFINITY;
  for (int x0 = 0; x0 < n; x0 += 4) {
    const int x = min(x0 + u, n - 1);
    const T* kp = kb + chain[x] * a.row;
    f32x4 s4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int y = 0; y < NI; ++y) s4 += qv[y] * load_w<T, 4>(kp, 4 * (j + 16 * y), a.D, true);
    float s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) s += __shfl_xor(s, off, 64);
    s *= a.sl2;
    top = fmaxf(top, s);
    if (j == 0 && x0 + u < n) score[x0 + u] = s;
  }
  wave_lds_sync();

  const Deal d = deal_slots(a.past, a.B, a.C, a.slots, -1, b);
  const int64_t rows = (int64_t)a.N * a.Hq;
  const int64_t pr0 = d.first * rows + (int64_t)i * a.Hq + h;
  for (int s = lane; s < d.count; s += 64) top = fmaxf(top, a.pm[pr0 + s * rows]);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  const float muse = top == -INFINITY ? 0.f : top;

  f32x4 acc[NI];
#pragma unroll
  for (int x = 0; x < NI; ++x) acc[x] = f32x4{0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  for (int s = u; s < d.count; s += 4) {
    const int64_t pr = pr0 + s * rows;
    const float w = exp2f(a.pm[pr] - muse);  // a split without keys: 0
    l += w * a.pl[pr];
#pragma unroll
    for (int x = 0; x < NI; ++x)
      acc[x] += load_w<float, 4>(a.po + pr * a.D, 4 * (j + 16 * x), a.D, true) * w;
  }
  for (int x = u; x < n; x += 4) {
    const float p = exp2f(score[x] - muse);
    const T* vp = vb + chain[x] * a.row;
    l += p;
#pragma unroll
    for (int y = 0; y < NI; ++y) acc[y] += load_w<T, 4>(vp, 4 * (j + 16 * y), a.D, true) * p;
  }
  l = group4_sum(l);
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int x = 0; x < NI; ++x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[x][e] = group4_sum(acc[x][e]) * inv;
    if (u == 0 && j + 16 * x < nch) store_vec4<T>(out + 4 * (j + 16 * x), acc[x]);
  }
  if (lane == 0) {
    if (a.m) a.m[si] = top == -INFINITY ? top : top * kLn2;
    if (a.l) a.l[si] = l;
  }
}

// ------------------------------------------------------------------- host --

struct Plan {
  int wave_rows, units, slots;
};

Plan make_plan(const CacheProblem& p) {
  const int64_t R = (int64_t)p.N * (p.Hq / p.Hkv);
  Plan x;
  x.wave_rows = R <= 16 ? 1 : R <= 32 ? 2 : 4;
  const int64_t rb = (R + 16 * x.wave_rows - 1) / (16 * x.wave_rows);
  x.units = (int)(rb * p.Hkv);
  const int64_t tiles = (int64_t)p.B * ((p.C + kTile - 1) / kTile);
  const int64_t deal = std::max<int64_t>(1, std::min<int64_t>(512 / x.units, tiles));
  x.slots = (int)(deal + p.B);
  return x;
}

}  // namespace

size_t cache_attn_bytes(const CacheProblem& p) {
  const Plan x = make_plan(p);
  return (size_t)x.slots * p.N * p.Hq * (p.D + 2) * sizeof(float);
}

hipError_t launch_cache_attn(const CacheProblem& p, const void* q, const void* k, const void* v,
                             void* out, float* m, float* l, void* ws, hipStream_t st) {
  const Plan x = make_plan(p);
  const int64_t prows = (int64_t)x.slots * p.N * p.Hq;
  AttnArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.m = m;
  a.l = l;
  a.po = static_cast<float*>(ws);
  a.pm = a.po + prows * p.D;
  a.pl = a.pm + prows;
  a.past = p.past;
  a.parents = p.parents;
  a.B = p.B;
  a.N = p.N;
  a.C = p.C;
  a.Hq = p.Hq;
  a.Hkv = p.Hkv;
  a.D = p.D;
  a.group = p.Hq / p.Hkv;
  a.R = p.N * a.group;
  a.slots = x.slots;
  a.units = x.units;
  a.wave_rows = x.wave_rows;
  a.seq = p.seq;
  a.row = p.row;
  a.head = p.head;
  a.sl2 = p.sl2;
  auto prefix = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(x.slots * x.units)), dim3(256), 0, st, a);
  };
  auto by_dim = [&](auto t) {
    using T = decltype(t);
    if (p.D <= 16) prefix(cache_prefix32_kernel<T, 1>);
    else if (p.D <= 32) prefix(cache_prefix32_kernel<T, 2>);
    else if (p.D <= 64) prefix(cache_prefix32_kernel<T, 4>);
    else if (p.D <= 96) prefix(cache_prefix32_kernel<T, 6>);
    else if (p.D <= 128) prefix(cache_prefix32_kernel<T, 8>);
    else prefix(cache_prefix32_kernel<T, 16>);
  };
  if (p.dtype == 1) by_dim(uint16_t{});
  else by_dim(float{});
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const unsigned blocks = (unsigned)(((int64_t)p.B * p.N * p.Hq + 3) / 4);
  auto merge = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, st, a); };
  auto merge_dim = [&](auto t) {
    using T = decltype(t);
    if (p.D <= 64) merge(cache_merge_kernel<T, 1>);
    else if (p.D <= 128) merge(cache_merge_kernel<T, 2>);
    else merge(cache_merge_kernel<T, 4>);
  };
  if (p.dtype == 1) merge_dim(uint16_t{});
  else merge_dim(float{});
  return hipGetLastError();
}

}  // namespace lc
