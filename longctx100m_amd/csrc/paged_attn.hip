// Attention of new tokens over a paged 8-bit cache (gfx950).
//
// Token i of sequence b, at row past_b + i of its cache, sees rows 0 .. past_b + i:
//   m = max s,  l = sum exp(s - m),  o = sum exp(s - m) v / l,  s = q k / sqrt(D),
// with k and v the e4m3 codes of the pages times their page's and head's scale.
// N tokens are R = N * Hq / Hkv query rows of a KV head.
//
// An e4m3 code has four significant bits and its scale is a power of two, so the
// product of both is a bf16 value exactly: the codes go to the bf16 matrix cores
// without any rounding, by one conversion (two values, with the scale) that
// costs less than the products.  fp32 queries and probabilities go in as three
// bf16 parts, x = x0 + x1 + x2, which hold all their 24 bits: an fp32 attention
// at a third of the bf16 rate instead of a sixteenth.
//
//   S^T = K Q^T     A = K, B = Q^T
//   O^T += V^T P^T  A = V^T, B = P^T, straight from the S^T accumulators
// with v_mfma_f32_16x16x32_bf16 (lane c = l % 16, g = l / 16: A row c, k-slots
// 8 g .. 8 g + 7; D rows 4 g + i of column c).  Which key a row of A is, and which
// dim or key a k-slot is, is free as long as both operands agree.  So a lane
// takes what lies together: 16 dims of key 16 (c / 4) + 4 mb + c % 4 of a 64-key
// tile, whose scores then are, for lane group g, those of keys 16 g .. 16 g + 15;
// and V^T is kept in that order ([dim][row] in a page), 16 keys of a dim in one
// 16-byte load.  Tiles go from memory to registers and from there to the
// products, with no LDS between.
#include "common.h"
#include "deal.h"
#include "e4m3.h"
#include "paged.h"
#include "tile128.h"
#include "tile32.h"

#include <algorithm>
#include <type_traits>

namespace lc {
namespace {

struct AttnArgs {
  PagedProblem p;
  const void* q;
  void* out;
  float *m, *l;
  // Partials, slot s of query row (token, head) at row * slots + s: D values, and
  // (m, l), m in log2 units.
  float* po;
  float2* ps;
  int2* deal;  // [B]: a sequence's first slot and its slots
  int group, R;
  int slots, units;  // units: workgroups of a slot
  int shift;         // log2 of a page's rows
  float sl2;
};

// Keys of a sequence: its past and its new tokens, as far as the page table goes.
__device__ __forceinline__ int keys_of(const AttnArgs& a, int b) {
  const int past = a.p.past[b];
  const int n = new_tokens(a.p.counts, a.p.N, b, past);
  return n > 0 ? (int)min((int64_t)past + n, (int64_t)a.p.width << a.shift) : 0;
}

__device__ __forceinline__ int64_t partial_row(const AttnArgs& a, int r, int hk, int slot) {
  return ((int64_t)(r / a.group) * a.p.Hq + hk * a.group + r % a.group) * a.slots + slot;
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Eight codes (two words) times a power of two.
__device__ __forceinline__ bf16x8 bf16_of(uint32_t lo, uint32_t hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The PARTS bf16 parts of eight fp32 values; what one rounds off is the next one's.
template <int PARTS>
__device__ __forceinline__ void split8(const f32x4& lo, const f32x4& hi, bf16x8 (&x)[PARTS]) {
  f32x4 a = lo, b = hi;
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    x[p] = pack_bf16x8(a, b);
    if (p + 1 < PARTS)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] -= (float)x[p][e];
        b[e] -= (float)x[p][4 + e];
      }
  }
}

// Bytes of a word that are NaN, as 0x80 each.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}
// The lowest n bytes of a word (n may be out of 0 .. 4).
__device__ __forceinline__ uint32_t low_bytes(int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << 8 * n) - 1u; }

// ------------------------------------------------------- a few query rows --

// Every wave holds all of the workgroup's 16 * NB rows and walks a run of the
// slot's tiles; the four waves meet in LDS.
// DP: head_dim, rounded up to 64, 128 or 256 unless EXACT.
template <int DP, bool EXACT, int NB, int PARTS>
__global__ __launch_bounds__(256, DP * PARTS > 192 ? 1 : 2) void paged_stream_kernel(AttnArgs a) {
  typedef typename std::conditional<PARTS == 1, uint16_t, float>::type T;
  constexpr int KJ = DP / 64, DB = DP / 16;  // 16-byte pieces of a key a lane takes; 16-dim blocks
  constexpr int W = 4, kRows = 16 * NB, kPitch = DP + 4;
  __shared__ __attribute__((aligned(16))) float part[W * kRows * kPitch];
  __shared__ float msm[W][kRows], lsm[W][kRows];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int slot = blockIdx.x / a.units;
  const int unit = blockIdx.x - slot * a.units;
  const Pool& pool = a.p.pool;
  const int hk = unit % pool.Hkv;
  const int rb = unit / pool.Hkv;
  const int D = EXACT ? DP : pool.D;
  Share s;
  if (!share_of([&](int b) { return keys_of(a, b); }, a.p.B, a.slots, a.deal, slot, s)) return;

  const int past = a.p.past[s.b];
  const int count = new_tokens(a.p.counts, a.p.N, s.b, past);
  const int32_t* table = a.p.table + (int64_t)s.b * a.p.width;
  // Tokens of this row block, and the rows that the last of them sees.
  const int first = rb * kRows / a.group, last = min((rb * kRows + kRows - 1) / a.group, count - 1);
  const int k1 = min(s.k1, past + last + 1);  // (no token: last < first, and nothing is walked)
  const int all = last >= first && k1 > s.k0 ? (k1 - s.k0 + 63) / 64 : 0;
  const int per = (all + W - 1) / W;
  const int t0 = s.k0 / 64 + min(wave * per, all), t1 = s.k0 / 64 + min((wave + 1) * per, all);

  // Rows of this lane: c of each 16; the keys they see.
  bf16x8 q[PARTS][NB][2 * KJ];
  int lim[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = rb * kRows + 16 * nb + c, i = r / a.group;
    const bool ok = r < a.R && i < count;
    lim[nb] = ok ? past + i + 1 : 0;
    const int64_t qi = ok ? ((int64_t)s.b * a.p.N + i) * a.p.Hq + hk * a.group + r % a.group : 0;
    const T* qp = static_cast<const T*>(a.q) + qi * D;
#pragma unroll
    for (int j = 0; j < 2 * KJ; ++j) {
      const int d = 64 * (j >> 1) + 16 * g + 8 * (j & 1);
      f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
      if (ok && (EXACT || d < D)) {
        lo = load_vec<T, 4>(qp + d);
        hi = load_vec<T, 4>(qp + d + 4);
      }
      bf16x8 x[PARTS];
      split8<PARTS>(lo, hi, x);
#pragma unroll
      for (int p = 0; p < PARTS; ++p) q[p][nb][j] = x[p];
    }
  }

  // The pages of the next 16 tiles: lane x has that of keys 16 x .. 16 x + 15 of
  // them, the page's two scales, and the row in it.
  int pages = -1;
  float kscale = 0.f, vscale = 0.f;
  auto look = [&](int t) {
    const int64_t key = 64 * (int64_t)t + 16 * lane;
    pages = -1;
    kscale = vscale = 1.f;  // (of no page: finite, its values are taken as zeros)
    if (key < k1) pages = page_of(table, a.p.width, pool.pages, key >> a.shift);
    if (pages >= 0) {
      const int64_t u = (int64_t)pages * pool.Hkv + hk;
      kscale = pool.ks[u];
      vscale = pool.vs[u];
    }
  };
  const int64_t head_bytes = (int64_t)D << a.shift;
  uint4 kr[4][KJ], vr[DB];
  auto base = [&](const uint8_t* p, int page) {
    return p + ((int64_t)max(page, 0) * pool.Hkv + hk) * head_bytes;
  };
  auto kload = [&](int t) {
    const int x = 4 * (t - t0 & 15) + (c >> 2);
    const int row = (64 * t + 16 * (c >> 2)) & ((1 << a.shift) - 1);
    const uint8_t* p = base(pool.k, __shfl(pages, x, 64)) + (row + (c & 3)) * D;
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        const int d = 64 * j + 16 * g;
        kr[mb][j] = *reinterpret_cast<const uint4*>(p + 4 * mb * D + (EXACT || d < D ? d : 0));
      }
  };
  auto vload = [&](int t) {
    const int x = 4 * (t - t0 & 15) + g;
    const int row = (64 * t + 16 * g) & ((1 << a.shift) - 1);
    const uint8_t* p = base(pool.v, __shfl(pages, x, 64)) + ((int64_t)c << a.shift) + row;
#pragma unroll
    for (int db = 0; db < DB; ++db)
      vr[db] = *reinterpret_cast<const uint4*>(p + ((int64_t)(EXACT || 16 * db < D ? 16 * db : 0) << a.shift));
  };

  f32x4 o[NB][DB];
  float mrow[NB], lsum[NB];  // running maximum (log2 units), lane-partial sum of p
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int db = 0; db < DB; ++db) o[nb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    mrow[nb] = -INFINITY;
    lsum[nb] = 0.f;
  }

  for (int t = t0; t < t1; ++t) {
    if ((t - t0 & 15) == 0) {
      look(t);
      kload(t);
      vload(t);
    }
    const int x = 4 * (t - t0 & 15);
    const float ks = __shfl(kscale, x + (c >> 2), 64);  // of the lane's K
    const float vs = __shfl(vscale, x + g, 64);         // of its V
    const int page = __shfl(pages, x + g, 64);
    f32x4 sc[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int mb = 0; mb < 4; ++mb) sc[nb][mb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KJ; ++j)
#pragma unroll
      for (int mb = 0; mb < 4; ++mb) {
        const bf16x8 k0 = bf16_of(kr[mb][j].x, kr[mb][j].y, ks), k1 = bf16_of(kr[mb][j].z, kr[mb][j].w, ks);
#pragma unroll
        for (int p = PARTS - 1; p >= 0; --p)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            sc[nb][mb] = mfma16x16x32(k0, q[p][nb][2 * j], sc[nb][mb]);
            sc[nb][mb] = mfma16x16x32(k1, q[p][nb][2 * j + 1], sc[nb][mb]);
          }
      }
    const bool more = t + 1 < t1 && (t + 1 - t0 & 15) != 0;
    if (more) kload(t + 1);

    // A tile that not every row sees wholly, or with a page that there is not.
    const bool edge = 64 * (t + 1) > past + 1 || __any(page < 0);
    bool strange = false;  // NaN among the values of such a tile
    if (edge) {
      const int left = page < 0 ? 0 : k1 - (64 * t + 16 * g);  // values that some row sees
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        vr[db].x &= low_bytes(left);
        vr[db].y &= low_bytes(left - 4);
        vr[db].z &= low_bytes(left - 8);
        vr[db].w &= low_bytes(left - 12);
        strange = strange || (nan_bytes(vr[db].x) | nan_bytes(vr[db].y) | nan_bytes(vr[db].z) | nan_bytes(vr[db].w));
      }
      strange = __any(strange);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int see = page < 0 ? 0 : lim[nb] - (64 * t + 16 * g);
#pragma unroll
        for (int mb = 0; mb < 4; ++mb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (4 * mb + i >= see) sc[nb][mb][i] = -INFINITY;
      }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float mx = -INFINITY;
#pragma unroll
      for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[nb][mb][i]);
      mx = group4_max(mx) * a.sl2;
      if (mx > mrow[nb]) {
        const float up = fast_exp2(mrow[nb] - mx);  // mrow = -inf: 0
        lsum[nb] *= up;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[nb][db] *= up;
        mrow[nb] = mx;
      }
      const float muse = mrow[nb] == -INFINITY ? 0.f : mrow[nb];
#pragma unroll
      for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = fast_exp2(fmaf(sc[nb][mb][i], a.sl2, -muse));
          lsum[nb] += p;
          sc[nb][mb][i] = p;
        }
    }
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2) {
      bf16x8 pb[NB][PARTS];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) split8<PARTS>(sc[nb][2 * k2], sc[nb][2 * k2 + 1], pb[nb]);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        uint32_t w0 = k2 ? vr[db].z : vr[db].x, w1 = k2 ? vr[db].w : vr[db].y;
        if (strange) {
          // A NaN must reach the rows that see it and no other: counted by itself.
          const uint32_t n0 = nan_bytes(w0), n1 = nan_bytes(w1);
          const uint32_t f0 = (n0 >> 7) * 0xffu, f1 = (n1 >> 7) * 0xffu;
          const bf16x8 is = bf16_of(f0 & 0x38383838u, f1 & 0x38383838u, 1.f);  // 1 where NaN
          w0 &= ~f0;
          w1 &= ~f1;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const f32x4 n = mfma16x16x32(is, pb[nb][0], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (n[i] > 0.f) o[nb][db][i] = NAN;
          }
        }
        const bf16x8 v = bf16_of(w0, w1, vs);
#pragma unroll
        for (int p = PARTS - 1; p >= 0; --p)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) o[nb][db] = mfma16x16x32(v, pb[nb][p], o[nb][db]);
      }
    }
    if (more) vload(t + 1);
  }

  // The waves' partials, brought to each row's maximum, meet in LDS.
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
    if (g == 0) msm[wave][16 * nb + c] = mrow[nb];
  __syncthreads();
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, msm[w][16 * nb + c]);
    const float f = mrow[nb] == -INFINITY ? 0.f : fast_exp2(mrow[nb] - M);
    const float lt = group4_sum(lsum[nb]) * f;
    if (g == 0) lsm[wave][16 * nb + c] = lt;
#pragma unroll
    for (int db = 0; db < DB; ++db)
      *reinterpret_cast<f32x4*>(part + (wave * kRows + 16 * nb + c) * kPitch + 16 * db + 4 * g) =
          mrow[nb] == -INFINITY ? f32x4{0.f, 0.f, 0.f, 0.f} : o[nb][db] * f;
  }
  __syncthreads();
  const int chunks = D / 4;  // of a row
  for (int it = threadIdx.x; it < kRows * chunks; it += 256) {
    const int rr = it / chunks, d = 4 * (it - rr * chunks);
    const int r = rb * kRows + rr;
    if (r >= a.R) break;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float L = 0.f, M = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      acc += *reinterpret_cast<const f32x4*>(part + (w * kRows + rr) * kPitch + d);
      L += lsm[w][rr];
      M = fmaxf(M, msm[w][rr]);
    }
    const int64_t pr = partial_row(a, r, hk, slot);
    *reinterpret_cast<f32x4*>(a.po + pr * D + d) = acc;
    if (d == 0) a.ps[pr] = make_float2(M, L);
  }
}

// ------------------------------------------------------------- the merge --

template <typename T>
__device__ __forceinline__ void store_vec4(T* p, const f32x4& r) {
  if constexpr (sizeof(T) == 4) store4(p, nullptr, r);
  else store4(nullptr, p, r);
}

// A wave per query row: lane 16 u + j holds 4-element chunks j, j + 16, .. of
// the head dim for the u-th of every four splits.
template <typename T, int NI>
__global__ __launch_bounds__(256) void paged_merge_kernel(AttnArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = lane & 15, u = lane >> 4;
  const int64_t row = 4 * (int64_t)blockIdx.x + wave;
  if (row >= (int64_t)a.p.B * a.p.N * a.p.Hq) return;
  const int h = (int)(row % a.p.Hq);
  const int64_t bi = row / a.p.Hq;
  const int b = (int)(bi / a.p.N), i = (int)(bi - (int64_t)b * a.p.N);
  const int D = a.p.pool.D, nch = D / 4;
  const bool there = i < new_tokens(a.p.counts, a.p.N, b, a.p.past[b]);
  const int2 deal = a.deal[b];
  const int splits = there ? deal.y : 0;
  const int64_t pr0 = ((int64_t)i * a.p.Hq + h) * a.slots + deal.x;
  float top = -INFINITY;
  for (int s = lane; s < splits; s += 64) top = fmaxf(top, a.ps[pr0 + s].x);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  const float muse = top == -INFINITY ? 0.f : top;
  f32x4 acc[NI];
#pragma unroll
  for (int x = 0; x < NI; ++x) acc[x] = f32x4{0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 4
  for (int s = u; s < splits; s += 4) {
    const int64_t pr = pr0 + s;
    const float2 st = a.ps[pr];
    const float w = exp2f(st.x - muse);  // a split without keys: 0
    l += w * st.y;
#pragma unroll
    for (int x = 0; x < NI; ++x)
      acc[x] += load_w<float, 4>(a.po + pr * D, 4 * (j + 16 * x), D, true) * w;
  }
  l = group4_sum(l);
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // NaN stays
  T* out = static_cast<T*>(a.out) + row * D;
#pragma unroll
  for (int x = 0; x < NI; ++x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[x][e] = group4_sum(acc[x][e]);
    if (u == 0 && j + 16 * x < nch) store_vec4<T>(out + 4 * (j + 16 * x), acc[x] * inv);
  }
  if (lane == 0) {
    const int64_t si = ((int64_t)b * a.p.Hq + h) * a.p.N + i;
    if (a.m) a.m[si] = top == -INFINITY ? top : top * kLn2;
    if (a.l) a.l[si] = l;
  }
}

// ------------------------------------------------------------------- host --

constexpr int64_t kWanted = 512;  // workgroups for the chip

struct Plan {
  int rows;  // of a workgroup
  int units, slots;
};

Plan make_plan(const PagedProblem& p) {
  const int64_t R = (int64_t)p.N * (p.Hq / p.pool.Hkv);
  const int64_t tiles = (int64_t)p.B * (((int64_t)p.width * p.pool.rows + kTile - 1) / kTile);
  Plan x;
  x.rows = 16;
  x.units = (int)((R + x.rows - 1) / x.rows * p.pool.Hkv);
  const int64_t slots = std::max<int64_t>(1, std::min<int64_t>(kWanted / x.units, tiles));
  x.slots = (int)(p.B > kTightBatch ? slots + p.B : std::max<int64_t>(slots, p.B > 1 ? p.B + slots / 2 : 1));
  return x;
}

}  // namespace

size_t paged_attn_bytes(const PagedProblem& p) {
  const Plan x = make_plan(p);
  return (size_t)x.slots * p.N * p.Hq * (p.pool.D + 2) * sizeof(float) + (size_t)p.B * sizeof(int2);
}

hipError_t launch_paged_attn(const PagedProblem& p, const void* q, void* out, float* m, float* l,
                             void* ws, hipStream_t st) {
  const Plan x = make_plan(p);
  const int64_t prows = (int64_t)x.slots * p.N * p.Hq;
  AttnArgs a;
  a.p = p;
  a.q = q;
  a.out = out;
  a.m = m;
  a.l = l;
  a.po = static_cast<float*>(ws);
  a.ps = reinterpret_cast<float2*>(a.po + prows * p.pool.D);
  a.deal = reinterpret_cast<int2*>(a.ps + prows);
  a.group = p.Hq / p.pool.Hkv;
  a.R = p.N * a.group;
  a.slots = x.slots;
  a.units = x.units;
  a.shift = __builtin_ctz((unsigned)p.pool.rows);
  a.sl2 = (float)(1.4426950408889634 / sqrt((double)p.pool.D));
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(x.slots * x.units)), dim3(256), 0, st, a);
  };
  auto by_dim = [&](auto parts) {
    constexpr int P = decltype(parts)::value;
    if (p.pool.D == 64) launch(paged_stream_kernel<64, true, 1, P>);
    else if (p.pool.D == 128) launch(paged_stream_kernel<128, true, 1, P>);
    else if (p.pool.D < 128) launch(paged_stream_kernel<128, false, 1, P>);
    else launch(paged_stream_kernel<256, false, 1, P>);
  };
  if (p.dtype == 1) by_dim(std::integral_constant<int, 1>{});
  else by_dim(std::integral_constant<int, 3>{});
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t rows = (int64_t)p.B * p.N * p.Hq;
  auto merge = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
  };
  auto merge_type = [&](auto t) {
    using T = decltype(t);
    if (p.pool.D <= 64) merge(paged_merge_kernel<T, 1>);
    else if (p.pool.D <= 128) merge(paged_merge_kernel<T, 2>);
    else merge(paged_merge_kernel<T, 4>);
  };
  if (p.dtype == 1) merge_type(uint16_t{});
  else merge_type(float{});
  return hipGetLastError();
}

}  // namespace lc
