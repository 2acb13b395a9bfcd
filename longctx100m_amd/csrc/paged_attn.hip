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
// at a third of the bf16 rate instead of a sixteenth.  bf16 queries round their
// probabilities to bf16, by 2^-8 at most each, the sum l not: outputs, which end in
// bf16, are off by 1.7 to 2.0e-3 instead of the 1.65e-3 of their own rounding.
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
  // Partials, part s of query row (token, head) at row * parts + s: D values, and
  // (m, l), m in log2 units.
  float* po;
  float2* ps;
  int2* deal;  // [B]: a sequence's first part and its parts
  int group, R;
  int slots, units;  // units: workgroups of a slot
  int parts;
  int shift;         // log2 of a page's rows
  bool direct;       // a slot is a whole sequence: results in place of partials
  bool early;        // and its table one run of pages, read beside its length
  float sl2;
};

// The rows before a sequence's new tokens, negative: none.  (A table has 2^30 rows at
// most, so more are as many.)
__device__ __forceinline__ int past_of(const int32_t* past, int b) { return min(past[b], 1 << 30); }

// Keys of a sequence: its past and its new tokens, as far as the page table goes.
__device__ __forceinline__ int keys_of(const AttnArgs& a, int b) {
  const int past = past_of(a.p.past, b);
  const int n = new_tokens(a.p.counts, a.p.N, b, past);
  return n > 0 ? (int)min((int64_t)past + n, (int64_t)a.p.width << a.shift) : 0;
}

// Tokens and heads of a block of query rows from r0 on: row r0 + x is token (r0 + x)
// / group.  One division for the block, then (x < 2^17, group <= 2^16) a float
// product that is off by less than half of 1 / group.
struct RowMap {
  int token0, rem, group;
  float inv;
  __device__ __forceinline__ RowMap(int r0, int group_) : group(group_) {
    token0 = __builtin_amdgcn_readfirstlane(r0 / group);
    rem = r0 - token0 * group;
    inv = 1.f / (float)group;
  }
  __device__ __forceinline__ int step(int x) const { return (int)(((float)(rem + x) + 0.5f) * inv); }
  __device__ __forceinline__ int token(int x) const { return token0 + step(x); }
  __device__ __forceinline__ int head(int x) const { return rem + x - step(x) * group; }
};

__device__ __forceinline__ int64_t partial_row(const AttnArgs& a, int r, int hk, int part) {
  return ((int64_t)(r / a.group) * a.p.Hq + hk * a.group + r % a.group) * a.parts + part;
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

// Values in a tile that not every row sees wholly go to the products without what
// no row sees (`left` of 16 keys are seen) and without NaN, which times a masked
// probability, a zero, would be NaN.  True: there was some, which the rows that
// see it get by patch_nan.
__device__ __forceinline__ bool clean_values(uint4& w, int left) {
  uint32_t x[4] = {w.x, w.y, w.z, w.w}, any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] &= low_bytes(left - 4 * i);
    const uint32_t n = nan_bytes(x[i]);
    x[i] &= ~((n >> 7) * 0xffu);
    any |= n;
  }
  w = make_uint4(x[0], x[1], x[2], x[3]);
  return any != 0;
}

template <typename T>
__device__ __forceinline__ void store_vec4(T* p, const f32x4& r) {
  if constexpr (sizeof(T) == 4) store4(p, nullptr, r);
  else store4(nullptr, p, r);
}

// 1 / l for a row's sum: 0 for a row that saw nothing, NaN for one that saw NaN.
__device__ __forceinline__ float inverse_sum(float l) { return l > 0.f ? 1.f / l : l; }

// The statistics of head h of token i of sequence b: its maximum in log2 units, and
// its sum.
__device__ __forceinline__ void store_stats(const AttnArgs& a, int b, int h, int i, float top, float l) {
  const int64_t si = ((int64_t)b * a.p.Hq + h) * a.p.N + i;
  if (a.m) a.m[si] = top == -INFINITY ? top : top * kLn2;
  if (a.l) a.l[si] = l;
}

// A run of 16 tiles (64 groups of 16 keys) of a walk, lane x with group x: its
// page (-1: none, or no key below `end`) and the page's scales.  The next run's
// are on their way during this one, the scales half a run after the pages that
// they follow from.
struct PageRun {
  int page, next;
  float ks, vs, nks, nvs;

  __device__ __forceinline__ void look(const AttnArgs& a, const int32_t* table, int t, int end) {
    const int64_t key = 64 * (int64_t)t + 16 * (threadIdx.x & 63);
    next = -1;
    if (key < end) next = page_of(table, a.p.width, a.p.pool.pages, key >> a.shift);
  }
  __device__ __forceinline__ void scales(const AttnArgs& a, int hk) {
    nks = nvs = 1.f;  // (of no page: finite, its values are taken as zeros)
    if (next >= 0) {
      const int64_t u = (int64_t)next * a.p.pool.Hkv + hk;
      nks = a.p.pool.ks[u];
      nvs = a.p.pool.vs[u];
    }
  }
  // Of a run that was looked up without an end: what lies at or behind it.
  __device__ __forceinline__ void cut(int end) {
    if (16 * (int)(threadIdx.x & 63) >= end) next = -1;
  }
  __device__ __forceinline__ void turn() {
    page = next;
    ks = nks;
    vs = nvs;
  }
};

// Calls put(n) for those of a row's dims dim(0) .. dim(N - 1) in which a value of the
// keys key0 .. key1 - 1 is NaN.
template <int N, typename Dim, typename Put>
__device__ __forceinline__ void patch_nan(const AttnArgs& a, const int32_t* table, int hk, int key0, int key1,
                                          const Dim& dim, const Put& put) {
  const Pool& pool = a.p.pool;
#pragma unroll 1
  for (int key = key0; key < key1; ++key) {
    const int page = page_of(table, a.p.width, pool.pages, key >> a.shift);
    if (page < 0) continue;
    const uint8_t* v = pool.v + ((((int64_t)page * pool.Hkv + hk) * pool.D) << a.shift) + (key & ((1 << a.shift) - 1));
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (dim(n) < pool.D && (v[(int64_t)dim(n) << a.shift] & 0x7f) == 0x7f) put(n);
  }
}

// ------------------------------------------------------- a few query rows --

// a, b of the lanes c and c ^ 8 of 16: the lower eight get (a, a of the other), the
// upper eight (b of the other, b).
__device__ __forceinline__ uint32_t ror8(uint32_t old, uint32_t x, bool upper) {
  return (uint32_t)(upper ? __builtin_amdgcn_update_dpp((int)old, (int)x, 0x128, 0xf, 0xc, false)
                          : __builtin_amdgcn_update_dpp((int)old, (int)x, 0x128, 0xf, 0x3, false));
}
__device__ __forceinline__ void swap_halves(uint4& a, uint4& b) {
  const uint4 t = a;
  a = make_uint4(ror8(a.x, b.x, true), ror8(a.y, b.y, true), ror8(a.z, b.z, true), ror8(a.w, b.w, true));
  b = make_uint4(ror8(b.x, t.x, false), ror8(b.y, t.y, false), ror8(b.z, t.z, false), ror8(b.w, t.w, false));
}

// 16 bytes that nobody else reads (NT), or that others find in L2.
template <bool NT>
__device__ __forceinline__ uint4 load16(const uint8_t* p) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  if constexpr (!NT) return *reinterpret_cast<const uint4*>(p);
  const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  return make_uint4(x[0], x[1], x[2], x[3]);
}

// Bound by the stream of the cache: one token over 262,143 rows of 8 heads of 128
// reads 537 MB in 91 us (5.9 TB/s), 32 sequences of 4,000 to 8,000 rows 398 MB in
// 71 (5.6); short ones by a chain of four memory latencies, kernel arguments,
// lengths, table, rows, of about a microsecond each (500 rows 8.5 us).  Every wave
// holds all of the workgroup's 16 rows and walks a run of the segment's tiles; the
// W waves meet in LDS.  (More rows are blocks of 16, whose second finds in L2 what
// the first has read: with 32 rows a wave 64 rows over 16,000 keys take 31 us for
// 28, over 131,072 106 for 115, and 64 of them do not fit the registers.)  A load of
// a wave should take whole cache lines: half a line at a time, its other half with
// the next load, costs a tenth of the stream.  So of a key of 128 bytes eight lanes
// take one half and eight the other, two loads take twice as many keys, and the
// lanes swap; the same for V in pages of 128 rows (VT = 2), a dim's line of which
// is two tiles' keys.
// DP: head_dim, rounded up to 64, 128 or 256 unless EXACT.
template <int DP, bool EXACT, int PARTS, int VT, bool NT, int W>
__global__ __launch_bounds__(64 * W, DP == 256 || W > 4 ? 1 : 2) void paged_stream_kernel(AttnArgs a) {
  typedef typename std::conditional<PARTS == 1, uint16_t, float>::type T;
  constexpr int KJ = DP / 64, DB = DP / 16;  // 16-byte pieces of a key a lane takes; 16-dim blocks
  constexpr int kRows = 16, kPitch = DP + 4;
  constexpr bool kLines = EXACT && DP == 128;
  static_assert(VT == 1 || EXACT, "two tiles of V at once");
  __shared__ __attribute__((aligned(16))) float part[W * kRows * kPitch];
  __shared__ float msm[W][kRows], lsm[W][kRows];
  // The parts of fp32 queries of 128 dims and more stay in LDS, a copy for all waves:
  // 48 registers fewer, with which two waves fit a SIMD (512 tokens of 32/8 heads of
  // 128 over 4,000 rows 125 us, 170 with the parts in registers; 64 over 16,001 69, 91).
  constexpr bool kShared = DP * PARTS > 192 && PARTS > 1;
  __shared__ __attribute__((aligned(16))) bf16x8 qs[kShared ? PARTS * 2 * KJ * 64 : 1];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slot = blockIdx.x / a.units;
  const int unit = blockIdx.x - slot * a.units;
  const Pool& pool = a.p.pool;
  const int hk = unit % pool.Hkv;
  const int rb = unit / pool.Hkv;
  const int D = EXACT ? DP : pool.D;
  PageRun run;
  if (a.early) run.look(a, a.p.table + (int64_t)slot * a.p.width, 0, 1 << 30);
  auto keys = [&](int b) { return keys_of(a, b); };
  for (Spans<64 * VT, decltype(keys)> s(keys, a.p.B, a.slots, a.direct, W, a.deal, slot); s.next();) {
    // (opaque: what follows from it is formed in each segment, not kept in registers)
    const int tid = opaque(threadIdx.x), lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int past = past_of(a.p.past, s.b);
    const int count = new_tokens(a.p.counts, a.p.N, s.b, past);
    const int32_t* table = a.p.table + (int64_t)s.b * a.p.width;
    // Tokens of this row block, and the rows that the last of them sees.
    const RowMap map(rb * kRows, a.group);
    const int first = map.token0, last = min(map.token(kRows - 1), count - 1);
    const int k1 = min(s.k1, past + last + 1);  // (no token: last < first, and nothing is walked)
    const int all = last >= first && k1 > s.k0 ? (k1 - s.k0 + 63) / 64 : 0;
    const int per = (all + W * VT - 1) / (W * VT) * VT;
    const int t0 = s.k0 / 64 + min(wave * per, all), t1 = s.k0 / 64 + min((wave + 1) * per, all);
    const int tb = a.early ? 0 : t0;     // the first tile of the page run
    const int clear = past + first + 1;  // keys that all rows see
    bool strange = false;                // NaN among the values that some rows see only
    if (a.early) run.cut(k1);
    else if (t0 < t1) run.look(a, table, t0, k1);

    // The lane's row: c; the keys it sees.
    const int qtok = map.token(c);
    const bool ok = rb * kRows + c < a.R && qtok < count;
    const int lim = ok ? past + qtok + 1 : 0;
    const int64_t qi = ok ? ((int64_t)s.b * a.p.N + qtok) * a.p.Hq + hk * a.group + map.head(c) : 0;
    const T* qp = static_cast<const T*>(a.q) + qi * D;
    auto qload = [&](int j, bf16x8 (&x)[PARTS]) {
      const int d = 64 * (j >> 1) + 16 * g + 8 * (j & 1);
      const bool on = ok && (EXACT || d < D);
      if constexpr (PARTS == 1) {
        x[0] = bf16x8{};
        if (on) x[0] = *reinterpret_cast<const bf16x8*>(qp + d);
      } else {
        f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
        if (on) {
          lo = load_vec<T, 4>(qp + d);
          hi = load_vec<T, 4>(qp + d + 4);
        }
        split8<PARTS>(lo, hi, x);
      }
    };
    bf16x8 q[kShared ? 1 : 2 * KJ][PARTS];
    if constexpr (kShared) {
      for (int j = wave; j < 2 * KJ; j += W) {
        bf16x8 x[PARTS];
        qload(j, x);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) qs[(j * PARTS + p) * 64 + lane] = x[p];
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int j = 0; j < 2 * KJ; ++j) qload(j, q[j]);
    }
    if (t0 < t1) run.scales(a, hk);

    const int64_t head_bytes = (int64_t)D << a.shift;
    const int page_mask = (1 << a.shift) - 1;
    uint4 kr[4][KJ], vr[VT][DB];
    auto base = [&](const uint8_t* p, int page) {
      return p + ((int64_t)max(page, 0) * pool.Hkv + hk) * head_bytes;
    };
    auto kload = [&](int t) {
      const int x = 4 * (t - tb & 15);
      if constexpr (kLines) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int gk = 2 * i + (c >> 2 & 1);
          const int row = 64 * t + 16 * gk & page_mask;
          const uint8_t* p =
              base(pool.k, __shfl(run.page, x + gk, 64)) + (row + (c & 3)) * D + 64 * (c >> 3) + 16 * g;
#pragma unroll
          for (int mb = 0; mb < 4; ++mb) kr[mb][i] = load16<NT>(p + 4 * mb * D);
        }
      } else {
        const int row = 64 * t + 16 * (c >> 2) & page_mask;
        const uint8_t* p = base(pool.k, __shfl(run.page, x + (c >> 2), 64)) + (row + (c & 3)) * D;
#pragma unroll
        for (int mb = 0; mb < 4; ++mb)
#pragma unroll
          for (int j = 0; j < KJ; ++j) {
            const int d = 64 * j + 16 * g;
            kr[mb][j] = load16<NT>(p + 4 * mb * D + (EXACT || d < D ? d : 0));
          }
      }
    };
    auto vload = [&](int t) {
      const int x = 4 * (t - tb & 15);
      if constexpr (VT == 2) {
        const uint8_t* p =
            base(pool.v, __builtin_amdgcn_readlane(run.page, x)) + 128 * (c & 7) + 64 * (c >> 3) + 16 * g;
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          vr[0][db] = load16<NT>(p + 128 * 16 * db);
          vr[1][db] = load16<NT>(p + 128 * (16 * db + 8));
        }
      } else {
        const int row = 64 * t + 16 * g & page_mask;
        const uint8_t* p = base(pool.v, __shfl(run.page, x + g, 64)) + ((int64_t)c << a.shift) + row;
#pragma unroll
        for (int db = 0; db < DB; ++db)
          vr[0][db] = load16<NT>(p + ((int64_t)(EXACT || 16 * db < D ? 16 * db : 0) << a.shift));
      }
    };

    f32x4 o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    float mrow = -INFINITY, lsum = 0.f;  // running maximum (log2 units), lane-partial sum of p

    if (t0 < t1) {
      run.turn();
      kload(t0);
      vload(t0);
      if (!a.early) run.look(a, table, t0 + 16, k1);
    }
    auto tile = [&](int t, auto sub) {
      constexpr int V = decltype(sub)::value;  // of the tiles whose values are here
      const int x = 4 * (t - tb & 15);
      const float ks = __shfl(run.ks, x + (c >> 2), 64);  // of the lane's K
      const float vs = __shfl(run.vs, x + g, 64);         // of its V
      const int page = __shfl(run.page, x + g, 64);
      if constexpr (kLines)
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) swap_halves(kr[mb][0], kr[mb][1]);
      if constexpr (VT == 2 && V == 0)
#pragma unroll
        for (int db = 0; db < DB; ++db) swap_halves(vr[0][db], vr[1][db]);
      f32x4 sc[4];
#pragma unroll
      for (int mb = 0; mb < 4; ++mb) sc[mb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        bf16x8 ql[PARTS], qh[PARTS];
        const int at = kShared ? opaque(lane) : 0;  // (read here in every tile)
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          ql[p] = kShared ? qs[(2 * j * PARTS + p) * 64 + at] : q[kShared ? 0 : 2 * j][p];
          qh[p] = kShared ? qs[((2 * j + 1) * PARTS + p) * 64 + at] : q[kShared ? 0 : 2 * j + 1][p];
        }
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) {
          const bf16x8 lo = bf16_of(kr[mb][j].x, kr[mb][j].y, ks), hi = bf16_of(kr[mb][j].z, kr[mb][j].w, ks);
#pragma unroll
          for (int p = PARTS - 1; p >= 0; --p) {
            sc[mb] = mfma16x16x32(lo, ql[p], sc[mb]);
            sc[mb] = mfma16x16x32(hi, qh[p], sc[mb]);
          }
        }
      }
      if (t + 1 < t1) {
        const int step = t + 1 - tb & 15;
        if (step == 0) {
          run.turn();
          run.look(a, table, t + 17, k1);
        } else if (step == 8 && !a.early) {
          run.scales(a, hk);
        }
        kload(t + 1);
      }

      // A tile that not every row sees wholly, or with a page that there is not.
      const bool edge = 64 * (t + 1) > clear;
      if (edge || __any(page < 0)) {
        const int left = page < 0 ? 0 : k1 - (64 * t + 16 * g);  // values that some row sees
        if (edge && last > first) {
#pragma unroll
          for (int db = 0; db < DB; ++db) strange |= clean_values(vr[V][db], left);
        } else {  // all rows see the same
          const uint32_t m[4] = {low_bytes(left), low_bytes(left - 4), low_bytes(left - 8), low_bytes(left - 12)};
#pragma unroll
          for (int db = 0; db < DB; ++db)
            vr[V][db] = make_uint4(vr[V][db].x & m[0], vr[V][db].y & m[1], vr[V][db].z & m[2], vr[V][db].w & m[3]);
        }
        const int see = page < 0 ? 0 : lim - (64 * t + 16 * g);
#pragma unroll
        for (int mb = 0; mb < 4; ++mb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (4 * mb + i >= see) sc[mb][i] = -INFINITY;
      }

      float mx = -INFINITY;
#pragma unroll
      for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[mb][i]);
      mx = group4_max(mx) * a.sl2;
      if (mx > mrow) {
        const float up = fast_exp2(mrow - mx);  // mrow = -inf: 0
        lsum *= up;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= up;
        mrow = mx;
      }
      const float muse = mrow == -INFINITY ? 0.f : mrow;
      float sum = 0.f;  // (a tile's by itself: over 18,000 keys 3e-7 from 64 bits, 1e-6 in one chain)
#pragma unroll
      for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = fast_exp2(fmaf(sc[mb][i], a.sl2, -muse));
          sum += p;
          sc[mb][i] = p;
        }
      lsum += sum;
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        bf16x8 pb[PARTS];
        split8<PARTS>(sc[2 * k2], sc[2 * k2 + 1], pb);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const bf16x8 v = bf16_of(k2 ? vr[V][db].z : vr[V][db].x, k2 ? vr[V][db].w : vr[V][db].y, vs);
#pragma unroll
          for (int p = PARTS - 1; p >= 0; --p) o[db] = mfma16x16x32(v, pb[p], o[db]);
        }
      }
    };
    for (int t = t0; t < t1; t += VT) {
      tile(t, std::integral_constant<int, 0>{});
      if constexpr (VT == 2)
        if (t + 1 < t1) tile(t + 1, std::integral_constant<int, 1>{});
      if (t + VT < t1) vload(t + VT);
    }
    if (__any(strange))
      patch_nan<4 * DB>(
          a, table, hk, max(64 * t0, clear & ~63), min(64 * t1, lim),
          [&](int n) { return 16 * (n >> 2) + 4 * g + (n & 3); }, [&](int n) { o[n >> 2][n & 3] = NAN; });

    // The waves' partials, brought to each row's maximum, meet in LDS.
    if (g == 0) msm[wave][c] = mrow;
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, msm[w][c]);
    const float f = mrow == -INFINITY ? 0.f : fast_exp2(mrow - top);
    lsum = group4_sum(lsum) * f;
    if (g == 0) lsm[wave][c] = lsum;
#pragma unroll
    for (int db = 0; db < DB; ++db)
      *reinterpret_cast<f32x4*>(part + (wave * kRows + c) * kPitch + 16 * db + 4 * g) =
          mrow == -INFINITY ? f32x4{0.f, 0.f, 0.f, 0.f} : o[db] * f;
    __syncthreads();
    const int chunks = D / 4;  // of a row
    for (int it = tid; it < kRows * chunks; it += 64 * W) {
      const int rr = it / chunks, d = 4 * (it - rr * chunks);
      if (rb * kRows + rr >= a.R) break;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      float L = 0.f, M = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        acc += *reinterpret_cast<const f32x4*>(part + (w * kRows + rr) * kPitch + d);
        L += lsm[w][rr];
        M = fmaxf(M, msm[w][rr]);
      }
      const int i = map.token(rr), h = hk * a.group + map.head(rr);
      if (a.direct) {
        const bool there = i < count;
        store_vec4(static_cast<T*>(a.out) + (((int64_t)s.b * a.p.N + i) * a.p.Hq + h) * D + d,
                   there ? acc * inverse_sum(L) : f32x4{0.f, 0.f, 0.f, 0.f});
        if (d == 0) store_stats(a, s.b, h, i, there ? M : -INFINITY, there ? L : 0.f);
      } else {
        const int64_t pr = ((int64_t)i * a.p.Hq + h) * a.parts + s.segment;
        *reinterpret_cast<f32x4*>(a.po + pr * D + d) = acc;
        if (d == 0) a.ps[pr] = make_float2(M, L);
      }
    }
    __syncthreads();  // the next segment's partials take their place
  }
}

// ------------------------------------------------------ many query rows --

// Bound by the products and the softmax beside them: 2,048 tokens of 32/8 heads of
// 128 behind 16,001 take 566 us, 1,007 TFLOP/s; a large library product reaches
// 1,172, and keeping the tile in 8 bits in LDS would have each wave convert all of
// it.  Eight waves of 32 rows share 64-key tiles of K and V^T, which the threads
// read from the pages as codes, 16 bytes at a time, one tile ahead, and write to
// LDS as bf16: converted once for 256 rows.  Iteration j issues the products of S^T
// for tile j + 1 and beside them, on the VALU, the softmax of tile j, then O^T +=
// V_j^T P_j^T; K runs one tile ahead of V, two buffers each, one barrier per tile.
// v_mfma_f32_32x32x16_bf16 (common.h): a lane's scores are those of row l % 32 with
// keys 8 (v / 4) + 4 h + v % 4, h = l / 32.  V^T rows are kept with each 16 keys in
// the order 0-3, 8-11, 4-7, 12-15, so that the eight of a lane half are one 16-byte
// read, and P^T needs no shuffle.  Chunks of 16 bytes of an LDS row of 128 bytes are
// XOR-swizzled by (row / 2) % 8, for reads without bank conflicts (tile128.h has
// the lane groups of a ds_read_b128).  A wave issues a VALU instruction in 8 cycles at
// best, two on a SIMD one in 4, and 128-dim rows leave registers for two: the products
// are 48% of the cycles, and neither earlier reads of LDS, nor half of the waves a phase
// behind, nor O's products beside the next tile's S changed more than 1%.
template <int D>
__global__ __launch_bounds__(512, 1) void paged_tile_kernel(AttnArgs a) {
  constexpr int BN = 64, RW = 8, KT = D / 16, DB = D / 32;  // products of S over the dims; 32-dim blocks
  constexpr int kTileB = BN * D * 2;
  constexpr int kStageK = 4 * D;  // threads that stage K: all 512, or (D = 64) the first half
  __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * kTileB];
  __shared__ uint32_t nan_s[RW];  // whether a wave has met NaN in V
  uint8_t* const kbuf = smem;
  uint8_t* const vbuf = smem + 2 * kTileB;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kc = lane & 31, hh = lane >> 5;
  const int slot = blockIdx.x / a.units;
  const int unit = blockIdx.x - slot * a.units;
  const Pool& pool = a.p.pool;
  const int hk = unit % pool.Hkv;
  const int rb = a.units / pool.Hkv - 1 - unit / pool.Hkv;  // the longest walks first
  Share s;
  if (!share_of([&](int b) { return keys_of(a, b); }, a.p.B, a.slots, a.deal, slot, s)) return;

  const int past = past_of(a.p.past, s.b);
  const int count = new_tokens(a.p.counts, a.p.N, s.b, past);
  const int32_t* table = a.p.table + (int64_t)s.b * a.p.width;
  constexpr int kRows = 32 * RW;
  // The keys of the workgroup's rows, and those of the wave's.
  const int first = rb * kRows / a.group, last = min((rb * kRows + kRows - 1) / a.group, count - 1);
  const int k1 = last >= first ? min(s.k1, past + last + 1) : s.k0;
  const int t0 = s.k0 / BN;
  const int ntiles = opaque(k1 > s.k0 ? (k1 - s.k0 + BN - 1) / BN : 0);
  const int wfirst = (rb * kRows + 32 * wave) / a.group;
  const int wlast = min((rb * kRows + 32 * wave + 31) / a.group, count - 1);
  const int wk1 = wlast >= wfirst ? min(k1, past + wlast + 1) : s.k0;
  const int nt_w = opaque(wk1 > s.k0 ? (wk1 - s.k0 + BN - 1) / BN : 0);
  const int clear = past + wfirst + 1;     // keys that every row of the wave sees
  const int all_clear = past + first + 1;  // and every row of the workgroup
  bool strange = false;                    // NaN among the values of tiles beyond

  const int r = rb * kRows + 32 * wave + kc, i = r / a.group;
  const bool ok = r < a.R && i < count;
  const int lim = ok ? past + i + 1 : 0;

  // Staging: a thread's piece of K is 16 dims of a row, of V 16 keys of a dim.
  const bool do_k = D == 128 || tid < kStageK, do_v = D == 128 || tid >= kStageK;
  const int krow = tid / (D / 16), kch = tid % (D / 16);
  const int vdim = (D == 128 ? tid : tid - kStageK) >> 2, vg = tid & 3;
  const int kg = __builtin_amdgcn_readfirstlane(krow >> 4) & 3;  // (uniform in the wave)
  const int64_t head_bytes = (int64_t)D << a.shift, page_bytes = pool.Hkv * head_bytes;
  const uint8_t* const kpages = pool.k + hk * head_bytes;
  const uint8_t* const vpages = pool.v + hk * head_bytes;
  const int page_mask = (1 << a.shift) - 1;
  const uint32_t kat = (krow & 15) * D + 16 * kch;                // in a page, from its group's first row
  const uint32_t vat = (vdim << a.shift) + (16 * vg & page_mask);  // from its tile's first row
  const int kdst = krow * 2 * D + 16 * ((2 * kch) ^ (D == 128 ? t128::swz(krow) : (krow >> 1) & 7));
  const int vdst = vdim * 128 + 16 * ((2 * vg) ^ ((vdim >> 1) & 7));
  PageRun run;
  uint4 kw, vw;
  float kscale, vscale;
  uint32_t gone = 0, gone_next = 0;  // of V's last two tiles, bit g: keys 16 g .. have no page
  // Tile j of K is read before that of V, and turns to a new run one tile earlier.
  auto kload = [&](int j) {
    if (j >= ntiles) return;
    if ((j & 15) == 8) run.scales(a, hk);
    const bool ahead = (j & 15) == 0;
    const int x = 4 * (j & 15) + kg;
    const int page = max(__builtin_amdgcn_readlane(ahead ? run.next : run.page, x), 0);
    kscale = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ahead ? run.nks : run.ks), x));
    const int row = BN * (t0 + j) + 16 * kg & page_mask;
    if (do_k) kw = *reinterpret_cast<const uint4*>(kpages + page * page_bytes + row * D + kat);
  };
  auto vload = [&](int j) {
    gone = gone_next;
    if (j >= ntiles) return;
    if ((j & 15) == 0) {
      run.turn();
      run.look(a, table, t0 + j + 16, k1);
    }
    const int x = 4 * (j & 15);
    const int row = BN * (t0 + j) & page_mask;
    // One page: its address and scale are the workgroup's (2% of the time of 2,048
    // tokens).
    if (page_mask >= BN - 1) {
      const int page = __builtin_amdgcn_readlane(run.page, x);
      gone_next = page < 0 ? 15 : 0;
      vscale = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(run.vs), x));
      if (do_v) vw = *reinterpret_cast<const uint4*>(vpages + max(page, 0) * page_bytes + row + vat);
    } else {
      gone_next = (uint32_t)(__ballot(run.page < 0) >> x) & 15u;
      vscale = __shfl(run.vs, x + vg, 64);
      const int page = max(__shfl(run.page, x + vg, 64), 0);
      if (do_v) vw = *reinterpret_cast<const uint4*>(vpages + page * page_bytes + row + vat);
    }
  };
  auto kwrite = [&](int j, auto parity) {  // parity: j % 2
    if (j >= ntiles || !do_k) return;
    uint8_t* const b = kbuf + decltype(parity)::value * kTileB;
    *reinterpret_cast<bf16x8*>(b + kdst) = bf16_of(kw.x, kw.y, kscale);
    *reinterpret_cast<bf16x8*>(b + (kdst ^ 16)) = bf16_of(kw.z, kw.w, kscale);
  };
  auto vwrite = [&](int j, auto parity) {
    constexpr int P = decltype(parity)::value;
    if (j >= ntiles) return;
    const bool edge = BN * (t0 + j) + BN > all_clear;
    if (edge || gone_next != 0) {
      const bool none = gone_next >> vg & 1;
      if (edge && do_v) strange |= clean_values(vw, none ? 0 : k1 - (BN * (t0 + j) + 16 * vg));
      else if (none) vw = make_uint4(0u, 0u, 0u, 0u);
    }
    if (!do_v) return;
    *reinterpret_cast<bf16x8*>(vbuf + P * kTileB + vdst) = bf16_of(vw.x, vw.z, vscale);
    *reinterpret_cast<bf16x8*>(vbuf + P * kTileB + (vdst ^ 16)) = bf16_of(vw.y, vw.w, vscale);
  };
  constexpr std::integral_constant<int, 0> even{};
  constexpr std::integral_constant<int, 1> odd{};
  if (ntiles > 0) {
    run.look(a, table, t0, k1);
    run.scales(a, hk);
    kload(0);
    kwrite(0, even);
    vload(0);
    vwrite(0, even);
    kload(1);
    kwrite(1, odd);
    vload(1);
    kload(2);
  }

  bf16x8 qreg[KT];  // lane: row r, dims 16 t + 8 hh .. + 7
  {
    const int64_t qi = ((int64_t)s.b * a.p.N + (ok ? i : 0)) * a.p.Hq + hk * a.group + r % a.group;
    const uint16_t* qrow = static_cast<const uint16_t*>(a.q) + qi * D;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      qreg[t] = *reinterpret_cast<const bf16x8*>(qrow + 16 * t + 8 * hh);
      if (!ok) qreg[t] = bf16x8{};
    }
  }
  const int koff = opaque(D == 128 ? t128::row_chunk_off(kc, hh) : kc * 128 + 16 * (hh ^ ((kc >> 1) & 7)));
  const int voff = opaque(kc * 128 + 16 * (hh ^ ((kc >> 1) & 7)));
  auto kread = [&](const uint8_t* kt, int n) {  // S step n: t = n / 2, mb = n % 2
    return *reinterpret_cast<const bf16x8*>(kt + (koff ^ 32 * (n >> 1)) + (n & 1) * 32 * 2 * D);
  };
  auto vread = [&](const uint8_t* vt, int n) {  // PV step n: u = n / DB, dims 32 (n % DB) ..
    return *reinterpret_cast<const bf16x8*>(vt + (voff ^ 32 * (n / DB)) + (n % DB) * 32 * 128);
  };

  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = f32x16{};
  float mrun = -INFINITY;  // log2 units, shared by the lanes l, l ^ 32
  float lsum = 0.f;        // lane-partial, relative to mrun

  auto scores_only = [&](const uint8_t* kt, f32x16 (&x)[2]) {
    bf16x8 A[2] = {kread(kt, 0), kread(kt, 1)};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 2 * KT; ++n) {
      x[n & 1] = mfma32x32x16(A[n & 1], qreg[n >> 1], n < 2 ? f32x16{} : x[n & 1]);
      if (n + 2 < 2 * KT) A[n & 1] = kread(kt, n + 2);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Tile j: klim, the lane's keys of it (less 4 hh); gone, bit g: no page for its
  // keys 16 g .. (both read if MASKED only).
  auto iteration = [&](auto masked_tag, auto next_tag, const uint8_t* kt, const uint8_t* vt, f32x16 (&sc)[2],
                       f32x16 (&sn)[2], int klim, uint32_t gone) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    constexpr bool NEXT = decltype(next_tag)::value;
    constexpr int S = 16;  // steps; 2 KT of them with a product
    constexpr int kEvery = S / (2 * KT);
    bf16x8 A[2], B[2], pb[4];
    if constexpr (NEXT) {
      A[0] = kread(kt, 0);
      A[1] = kread(kt, 1);
    }
    float pmax = -INFINITY, muse = 0.f, sum[2] = {0.f, 0.f};  // (sum: as in the streaming form)
    auto argument = [&](int e) { sc[e >> 4][e & 15] = fmaf(sc[e >> 4][e & 15], a.sl2, -muse); };
    auto exponential = [&](int e) { sc[e >> 4][e & 15] = fast_exp2(sc[e >> 4][e & 15]); };
    auto add = [&](int e) { sum[e & 1] += sc[e >> 4][e & 15]; };
    auto pack = [&](int mb) {  // the B operands of keys 32 mb .. 32 mb + 31
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int e = 8 * u;
        pb[2 * mb + u] = pack_bf16x8(f32x4{sc[mb][e], sc[mb][e + 1], sc[mb][e + 2], sc[mb][e + 3]},
                                     f32x4{sc[mb][e + 4], sc[mb][e + 5], sc[mb][e + 6], sc[mb][e + 7]});
      }
    };
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int st = 0; st < S; ++st) {
      if constexpr (NEXT)
        if (st % kEvery == 0) {
          const int n = st / kEvery;
          sn[n & 1] = mfma32x32x16(A[n & 1], qreg[n >> 1], n < 2 ? f32x16{} : sn[n & 1]);
          if (n + 2 < 2 * KT) A[n & 1] = kread(kt, n + 2);
        }
      if (st < 4) {  // the maximum, 8 scores per step
#pragma unroll
        for (int e = 8 * st; e < 8 * st + 8; ++e) {
          const int mb = e >> 4, v = e & 15;
          if constexpr (MASKED)
            if (32 * mb + 8 * (v >> 2) + (v & 3) >= klim || (gone >> (2 * mb + (v >> 3)) & 1)) sc[mb][v] = -INFINITY;
          pmax = fmaxf(pmax, sc[mb][v]);
        }
      }
      if (st == 7) {
        const float mx = xor32_max(pmax) * a.sl2;
        if (__any(mx > mrun)) {
          const float alpha = mx > mrun ? fast_exp2(mrun - mx) : 1.f;  // mrun = -inf: 0
          mrun = fmaxf(mrun, mx);
          lsum *= alpha;
#pragma unroll
          for (int d = 0; d < DB; ++d) o[d] *= alpha;
        }
        muse = mrun == -INFINITY ? 0.f : mrun;
      }
      // Probabilities, 4 per step, each in three steps, argument, exponential and sum, so
      // that nothing waits for the instruction before it.
      if (st >= 7)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (st >= 8) exponential(4 * (st - 8) + k);
          if (st < 15) argument(4 * (st - 7) + k);
          if (st >= 9) add(4 * (st - 9) + k);
        }
      if (st == 12) pack(0);
      if (st == 14) B[0] = vread(vt, 0);
      if (st == 15) B[1] = vread(vt, 1);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int k = 28; k < 32; ++k) add(k);
    pack(1);
    lsum += sum[0] + sum[1];
#pragma unroll
    for (int n = 0; n < 4 * DB; ++n) {
      o[n % DB] = mfma32x32x16(B[n & 1], pb[n / DB], o[n % DB]);
      if (n + 2 < 4 * DB) B[n & 1] = vread(vt, n + 2);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Step j of the workgroup: tiles j + 2 of K and j + 1 of V to LDS, the next ones on
  // their way.  Returns tile j's groups without a page.
  auto stage = [&](int j, auto parity) {
    constexpr int P = decltype(parity)::value;  // j % 2
    __syncthreads();
    kwrite(j + 2, parity);
    vwrite(j + 1, std::integral_constant<int, P ^ 1>{});
    const uint32_t none = gone;
    vload(j + 2);
    kload(j + 3);
    return none;
  };
  auto masked = [&](int j, auto parity, auto next, f32x16 (&sc)[2], f32x16 (&sn)[2], uint32_t none) {
    constexpr int P = decltype(parity)::value;
    iteration(std::true_type{}, next, kbuf + (P ^ 1) * kTileB, vbuf + P * kTileB, sc, sn,
              opaque(lim - BN * (t0 + j) - 4 * hh), none);
  };
  auto step = [&](int j, auto parity, f32x16 (&sc)[2], f32x16 (&sn)[2]) {
    constexpr int P = decltype(parity)::value;
    const uint32_t none = stage(j, parity);
    if (BN * (t0 + j) + BN > clear || none != 0)
      masked(j, parity, std::true_type{}, sc, sn, none);
    else
      iteration(std::false_type{}, std::true_type{}, kbuf + (P ^ 1) * kTileB, vbuf + P * kTileB, sc, sn, 0, 0);
  };
  f32x16 sa[2], sb[2];
  __syncthreads();
  int j = 0;
  if (nt_w > 0) {
    scores_only(kbuf, sa);
    for (; j + 2 < nt_w; j += 2) {
      step(j, even, sa, sb);
      step(j + 1, odd, sb, sa);
    }
    if (j + 1 < nt_w) {
      step(j, even, sa, sb);
      ++j;
      masked(j, odd, std::false_type{}, sb, sa, stage(j, odd));
    } else {
      masked(j, even, std::false_type{}, sa, sb, stage(j, even));
    }
    ++j;
  }
  for (; j < ntiles; ++j) {  // what the other waves' rows see beyond
    if (j & 1) stage(j, odd);
    else stage(j, even);
  }

  const uint64_t any = __ballot(strange);
  if (lane == 0) nan_s[wave] = any != 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < RW; ++w) strange |= nan_s[w] != 0;
  if (strange)
    patch_nan<16 * DB>(
        a, table, hk, max(s.k0, all_clear & ~(BN - 1)), min(k1, lim),
        [&](int n) { return 32 * (n >> 4) + 8 * ((n & 15) >> 2) + 4 * hh + (n & 3); },
        [&](int n) { o[n >> 4][n & 15] = NAN; });
  const float l = xor32_sum(lsum);
  if (r >= a.R) return;
  const float f = a.direct ? (ok ? inverse_sum(l) : 0.f) : 1.f;
  const bool nothing = a.direct ? !ok : mrun == -INFINITY;
  const int64_t pr = partial_row(a, r, hk, slot);
  uint16_t* out = static_cast<uint16_t*>(a.out) + (((int64_t)s.b * a.p.N + i) * a.p.Hq + hk * a.group + r % a.group) * D;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f32x4 x = f32x4{o[d][4 * w], o[d][4 * w + 1], o[d][4 * w + 2], o[d][4 * w + 3]} * f;
      if (nothing) x = f32x4{0.f, 0.f, 0.f, 0.f};
      const int at = 32 * d + 8 * w + 4 * hh;
      if (a.direct) store4(nullptr, out + at, x);
      else *reinterpret_cast<f32x4*>(a.po + pr * D + at) = x;
    }
  if (hh == 0) {
    if (a.direct) store_stats(a, s.b, hk * a.group + r % a.group, i, ok ? mrun : -INFINITY, ok ? l : 0.f);
    else a.ps[pr] = make_float2(mrun, l);
  }
}

// ------------------------------------------------------------- the merge --

// WPR waves per query row, its parts dealt over them: lane 16 u + j holds 4-element
// chunks j, j + 16, .. of the head dim for the u-th of every four parts.
template <typename T, int NI, int WPR>
__global__ __launch_bounds__(256) void paged_merge_kernel(AttnArgs a) {
  constexpr int kRows = 4 / WPR;  // of a workgroup
  __shared__ float top_s[4], l_s[4];
  __shared__ f32x4 acc_s[4][16 * NI];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = lane & 15, u = lane >> 4, w0 = wave % WPR;
  const int64_t row = kRows * (int64_t)blockIdx.x + wave / WPR;
  if (row >= (int64_t)a.p.B * a.p.N * a.p.Hq) return;  // (WPR = 4: nobody)
  const int h = (int)(row % a.p.Hq);
  const int64_t bi = row / a.p.Hq;
  const int b = (int)(bi / a.p.N), i = (int)(bi - (int64_t)b * a.p.N);
  const int D = a.p.pool.D, nch = D / 4;
  const bool there = i < new_tokens(a.p.counts, a.p.N, b, a.p.past[b]);
  const int2 deal = a.deal[b];
  const int parts = there ? deal.y : 0;
  const int64_t pr0 = ((int64_t)i * a.p.Hq + h) * a.parts + deal.x;
  float top = -INFINITY;
  for (int s = 64 * w0 + lane; s < parts; s += 64 * WPR) top = fmaxf(top, a.ps[pr0 + s].x);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if constexpr (WPR > 1) {
    if (lane == 0) top_s[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WPR; ++w) top = fmaxf(top, top_s[w]);
  }
  const float muse = top == -INFINITY ? 0.f : top;
  f32x4 acc[NI];
#pragma unroll
  for (int x = 0; x < NI; ++x) acc[x] = f32x4{0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 4
  for (int s = 4 * w0 + u; s < parts; s += 4 * WPR) {
    const int64_t pr = pr0 + s;
    const float2 st = a.ps[pr];
    const float w = exp2f(st.x - muse);  // a part without keys: 0
    l += w * st.y;
#pragma unroll
    for (int x = 0; x < NI; ++x)
      acc[x] += load_w<float, 4>(a.po + pr * D, 4 * (j + 16 * x), D, true) * w;
  }
  l = group4_sum(l);
#pragma unroll
  for (int x = 0; x < NI; ++x)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[x][e] = group4_sum(acc[x][e]);
  if constexpr (WPR > 1) {
    if (u == 0)
#pragma unroll
      for (int x = 0; x < NI; ++x) acc_s[wave][j + 16 * x] = acc[x];
    if (lane == 0) l_s[wave] = l;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < WPR; ++w) {
      l += l_s[w];
#pragma unroll
      for (int x = 0; x < NI; ++x) acc[x] += acc_s[w][j + 16 * x];
    }
  }
  const float inv = inverse_sum(l);
  T* out = static_cast<T*>(a.out) + row * D;
#pragma unroll
  for (int x = 0; x < NI; ++x)
    if (u == 0 && j + 16 * x < nch) store_vec4<T>(out + 4 * (j + 16 * x), acc[x] * inv);
  if (lane == 0) store_stats(a, b, h, i, top, l);
}

// ------------------------------------------------------------------- host --

constexpr int64_t kWanted = 512;  // workgroups of the streaming form for the chip
constexpr int64_t kWantedTiled = 256;
constexpr int64_t kShort = 16;  // tiles of a sequence that are not split over workgroups

// Many rows go by tiles that a workgroup shares once all blocks of 16 rows together
// would read more than this, at the tables' width; up to there, and up to kFewRows
// rows a KV head, each block reads the cache by itself.  Later ones read it from L2 where
// KV heads are a multiple of eight: a head's blocks lie that many workgroups apart, which
// go to the XCDs in turn.  Measured with 32/8 heads only (blocks of 16 against tiles,
// us).  Of 128: 24 tokens over 2,000 keys (25 MB) 18.4
// and 21.4, 64 over 500 (18 MB) 12.7 and 20.6, 64 over 4,000 (133 MB) 27.3 and 31.9, 32
// over 16,000 (263 MB) 38.5 and 31.8, 256 over 8,000 (1.1 GB) 98 and 63; eight
// sequences' 64 over 500 (148 MB) 27 and 36, 32 over 2,000 (266 MB) 41 and 33.  Of 64: 64
// tokens over 8,000 (132 MB) 22 and 26, 128 over 16,000 (529 MB) 52 and 44.  8 tokens over
// 131,072 keys (537 MB) 78 and 87.  Around the limit either is up to a sixth behind.
constexpr int64_t kBlockBytes = 160 << 20;
constexpr int64_t kFewRows = 48;

// Query rows from which a wave each is enough for the merge.
constexpr int64_t kManyRows = 1024;

// Of the tiled form one workgroup runs on a CU, so those beyond 256 wait for a second
// round, and slots are whole: the time goes in steps.  32/8 heads of 128 behind 16,001:
// 1,024 tokens (two slots) 331 us, 1,088 488, 1,536 502, 2,048 (256 workgroups) 565, 2,112 956,
// 3,000 1,003, 4,096 1,127.
struct Plan {
  bool tiled;
  int rows;  // of a workgroup
  int tile;  // keys by which sequences are dealt out
  int waves;
  int units, slots, parts;  // parts: 0, results without a merge
};

Plan make_plan(const PagedProblem& p) {
  const int64_t R = (int64_t)p.N * (p.Hq / p.pool.Hkv);
  Plan x;
  const int64_t reads = (R + 15) / 16 * p.B * p.width * p.pool.rows * p.pool.Hkv * p.pool.D * 2;
  x.tiled = p.dtype == 1 && (p.pool.D == 64 || p.pool.D == 128) && R > kFewRows && reads > kBlockBytes;
  x.rows = x.tiled ? 256 : 16;
  x.tile = !x.tiled && p.pool.rows == 128 && (p.pool.D == 64 || p.pool.D == 128) ? 128 : 64;
  x.units = (int)((R + x.rows - 1) / x.rows * p.pool.Hkv);
  const int64_t each = ((int64_t)p.width * p.pool.rows + x.tile - 1) / x.tile;  // tiles of a sequence
  const int64_t want = (x.tiled ? kWantedTiled : kWanted) / x.units;
  x.waves = 8;
  if (x.tiled) {
    const int64_t slots = std::max<int64_t>(1, std::min<int64_t>(want, p.B * each));
    x.slots = slots == 1           ? p.B
              : p.B > kTightBatch ? (int)slots + p.B
                                  : (int)std::max<int64_t>(slots, p.B > 1 ? p.B + slots / 2 : 1);
    x.parts = x.slots == p.B ? 0 : x.slots;
    return x;
  }
  if (each <= kShort || want <= 1) {
    x.waves = want <= p.B || p.dtype == 0 || (p.pool.D != 64 && p.pool.D != 128) ? 4 : 8;
    x.slots = p.B;
    x.parts = 0;
  } else {
    x.waves = 4;
    x.slots = (int)std::max<int64_t>(1, std::min<int64_t>(want, (p.B * each + x.waves - 1) / x.waves));
    x.parts = x.slots + p.B;
  }
  return x;
}

}  // namespace

size_t paged_attn_bytes(const PagedProblem& p) {
  return (size_t)make_plan(p).parts * p.N * p.Hq * (p.pool.D + 2) * sizeof(float) + (size_t)p.B * sizeof(int2);
}

hipError_t launch_paged_attn(const PagedProblem& p, const void* q, void* out, float* m, float* l,
                             void* ws, hipStream_t st) {
  const Plan x = make_plan(p);
  const int64_t prows = (int64_t)x.parts * p.N * p.Hq;
  AttnArgs a;
  a.p = p;
  a.q = q;
  a.out = out;
  a.m = m;
  a.l = l;
  a.direct = x.parts == 0;
  a.early = a.direct && !x.tiled && (int64_t)p.width * p.pool.rows <= 1024;
  a.parts = x.parts;
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
    hipLaunchKernelGGL(kernel, dim3((unsigned)(x.slots * x.units)), dim3(64 * x.waves), 0, st, a);
  };
  // The cache is read once: past L2, also what sequences of a common prefix share.
  const bool once = x.units == p.pool.Hkv;
  auto by_dim = [&](auto parts, auto nt) {
    constexpr int P = decltype(parts)::value;
    constexpr bool NT = decltype(nt)::value;
    const bool two = x.tile == 128;
    auto by_waves = [&](auto d, auto vt) {
      constexpr int DP = decltype(d)::value, VT = decltype(vt)::value;
      if constexpr (P == 1)
        if (x.waves == 8) return launch(paged_stream_kernel<DP, true, P, VT, NT, 8>);
      launch(paged_stream_kernel<DP, true, P, VT, NT, 4>);
    };
    auto by_pages = [&](auto d) {
      if (two) by_waves(d, std::integral_constant<int, 2>{});
      else by_waves(d, std::integral_constant<int, 1>{});
    };
    if (p.pool.D == 64) by_pages(std::integral_constant<int, 64>{});
    else if (p.pool.D == 128) by_pages(std::integral_constant<int, 128>{});
    else if (p.pool.D < 128) launch(paged_stream_kernel<128, false, P, 1, NT, 4>);
    else launch(paged_stream_kernel<256, false, P, 1, NT, 4>);
  };
  auto by_reads = [&](auto parts) {
    if (once) by_dim(parts, std::true_type{});
    else by_dim(parts, std::false_type{});
  };
  if (x.tiled && p.pool.D == 64) launch(paged_tile_kernel<64>);
  else if (x.tiled) launch(paged_tile_kernel<128>);
  else if (p.dtype == 1) by_reads(std::integral_constant<int, 1>{});
  else by_reads(std::integral_constant<int, 3>{});
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.direct) return e;
  const int64_t rows = (int64_t)p.B * p.N * p.Hq;
  auto merge = [&](auto kernel, int each) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)((rows + each - 1) / each)), dim3(256), 0, st, a);
  };
  auto merge_dim = [&](auto t, auto ni) {
    using T = decltype(t);
    constexpr int NI = decltype(ni)::value;
    if (rows < kManyRows) merge(paged_merge_kernel<T, NI, 4>, 1);
    else merge(paged_merge_kernel<T, NI, 1>, 4);
  };
  auto merge_type = [&](auto t) {
    if (p.pool.D <= 64) merge_dim(t, std::integral_constant<int, 1>{});
    else if (p.pool.D <= 128) merge_dim(t, std::integral_constant<int, 2>{});
    else merge_dim(t, std::integral_constant<int, 4>{});
  };
  if (p.dtype == 1) merge_type(uint16_t{});
  else merge_type(float{});
  return hipGetLastError();
}

}  // namespace lc
