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
//   2. cache_merge_kernel, one or four waves per row, follows the row's chain,
//      takes its few keys with fp32 dot products and merges them with the
//      partials.
// Neither multiplies a row of the cache by a masked probability (a tile that the
// past ends in is filled up with rows of zeros), so what stands in a row that a
// token does not see cannot reach it, whatever it is.
//
// The lengths are known on the device only.  The host fixes the number of
// split slots (and with it the workspace); each workgroup reads the lengths
// and finds its sequence and key range: a slot holds `per` tiles, the fewest
// with which the slots suffice for all sequences, so a batch of unequal
// lengths loads the chip evenly.
#include "common.h"
#include "cache.h"
#include "kernels.h"
#include "stream_tile.h"
#include "tile128.h"
#include "tile32.h"

#include <algorithm>
#include <type_traits>

namespace lc {
namespace {

constexpr int kTile = 64;  // keys by which the past is dealt out

// What the rows of a V tile behind the past hold: their probabilities are zeros,
// but the past's last row again would make 0 * inf of an infinity in it.
__device__ const uint4 kZeroRow = {0u, 0u, 0u, 0u};

struct AttnArgs {
  const void *q, *k, *v;
  void* out;
  float *m, *l;
  // Partials, slot s of query row (token, head) at row * slots + s: D values, and
  // (m, l), m in log2 units.
  float* po;
  float2* ps;
  int2* deal;  // [B]: a sequence's first slot and its slots
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

__device__ __forceinline__ int wave_sum_i(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// ceil(t / per) for 0 <= t < 2^24, inv = 1 / per: the product is off by at most
// one.
__device__ __forceinline__ int slots_for(int t, int per, float inv) {
  const int q = (int)((float)t * inv);
  const int r = t - q * per;
  return q + (r > 0) + (r > per);
}

// Sequences up to which the slots are dealt as tightly as possible.
constexpr int kTightBatch = 64;

// Tiles of a slot.  One sequence: its share.  Up to kTightBatch: the 64 lanes
// try 63 sizes from an even share of all tiles to five times it, and the longest
// sequence's tiles, with which one slot a sequence is enough; the smallest
// size whose slots suffice is taken.  More sequences have B slots beyond the
// even shares, and ceil(tiles / per) adds less than one each.
__device__ __forceinline__ int slot_tiles(const int32_t* past, int B, int C, int slots) {
  const int lane = threadIdx.x & 63;
  if (B == 1) return (past_tiles(past[0], C) + slots - 1) / slots;
  if (B > kTightBatch) {
    int total = 0;
    for (int b0 = 0; b0 < B; b0 += 64)
      total += wave_sum_i(b0 + lane < B ? past_tiles(past[b0 + lane], C) : 0);
    return (total + slots - B - 1) / (slots - B);
  }
  const int mine = lane < B ? past_tiles(past[lane], C) : 0;
  int most = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) most = max(most, __shfl_xor(most, off, 64));
  const int even = (wave_sum_i(mine) + slots - 1) / slots;
  const int size = lane == 63 ? most : even + (int)((int64_t)even * lane / 16);
  const float inv = 1.f / (float)size;
  int n = 0;
  for (int b = 0; b < B; ++b) n += slots_for(__builtin_amdgcn_readlane(mine, b), size, inv);
  const uint64_t fits = __ballot(n <= slots);  // the last lane's does
  return __builtin_amdgcn_readlane(size, __ffsll((unsigned long long)fits) - 1);
}

// The key range of a workgroup.
struct Share {
  int b, k0, k1;  // keys k0 .. k1 - 1 of sequence b (none: k0 == k1)
};
// Finds the share of a slot; false: it has none.  The first workgroup leaves
// every sequence's slots for the merge.
__device__ __forceinline__ bool share_of(const AttnArgs& a, int slot, Share& s) {
  const int lane = threadIdx.x & 63;
  const int per = slot_tiles(a.past, a.B, a.C, a.slots);
  const float inv = 1.f / (float)per;
  int first = 0, at = -1;  // of sequence at
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    const int n = b < a.B ? slots_for(past_tiles(a.past[b], a.C), per, inv) : 0;
    const int end = base + wave_scan(n);
    if (blockIdx.x == 0 && threadIdx.x < 64 && b < a.B) a.deal[b] = make_int2(end - n, n);
    const uint64_t who = __ballot(slot < end && slot >= end - n);
    if (who) {
      const int x = __ffsll((unsigned long long)who) - 1;
      at = b0 + x;
      first = __builtin_amdgcn_readlane(end - n, x);
    }
    base = __builtin_amdgcn_readlane(end, 63);
  }
  if (at < 0) return false;
  s.b = __builtin_amdgcn_readfirstlane(at);
  const int rows = past_rows(a.past[s.b], a.C);
  s.k0 = __builtin_amdgcn_readfirstlane(min((slot - first) * per * kTile, rows));
  s.k1 = __builtin_amdgcn_readfirstlane(min(rows - s.k0, per * kTile)) + s.k0;
  return true;
}

// Where the partial of query row r of KV head hk goes.
__device__ __forceinline__ int64_t partial_row(const AttnArgs& a, int r, int hk, int slot) {
  return ((int64_t)(r / a.group) * a.Hq + hk * a.group + r % a.group) * a.slots + slot;
}

// ------------------------------------------------- the past, fp32 products --

// fp32, precise bf16 and other head dims, on the fp32 matrix cores (13 tokens of
// 2 x 9/3 heads of 64 over 2,047 keys: 11 us).
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
    const int64_t pr = partial_row(a, row, hk, slot);
    *reinterpret_cast<f32x4*>(a.po + pr * a.D + d) = acc;
    if (d == 0) a.ps[pr] = make_float2(mt, ls);
  }
}

// ------------------------------------------- the past, bf16, a few rows --

// Few query rows: bound by the stream of the cache.  Every wave holds all of
// the workgroup's 16 * NB rows (Q^T in registers, the B operand) and takes its
// own 8 KB tiles of K, straight into registers as the A operand of S^T = K Q^T,
// and of V, through LDS for the transposed reads of O^T += V^T P^T; both one
// tile ahead.  With 64 rows there are registers for one K tile: the next is
// read once the scores are there.  The four waves of a workgroup take the tiles
// of their split in turn and meet in LDS.  Probabilities go to the products in
// bf16, relative to the row's exact running maximum in the wave (their sum stays
// fp32): 1.74e-3 from 64 bits at 8 tokens over 500 keys, the output's rounding alone
// 1.67e-3.  (2,048 workgroups of one wave, the
// slots of a KV head next to each other, gain with up to 16 rows and 262,000 keys
// alone, 174 us against 193 for one token; up to 120,000 keys the merge of their
// partials costs what they gain, and with 32 rows they gain nothing.)
// NT, rows of 128 dims that one workgroup reads once: non-temporal loads, which
// leave the partials in L2 for the merge: 53 us in all against 56 at 60,000 keys
// and 4 tokens, 194 against 200 at 262,000 (5.7 TB/s).  Rows of 64 are one cache
// line of which each load takes half: 30.1 us in all against 35.0 at 60,000 keys
// and 8 tokens, 112 against 118 at 262,000 and 4 (5.0 TB/s).  Two row blocks
// find in L2 what the other has read.
template <int D, int NB, bool NT>
__global__ __launch_bounds__(256, 2) void cache_stream_kernel(AttnArgs a) {
  using C = DecodeTile<D>;
  constexpr int TK = C::TK, MB = C::MB, KS = C::KS, DB = C::DB;
  constexpr int W = 4;  // waves
  constexpr int kRows = 16 * NB;
  constexpr int kStages = 2;
  constexpr int kPitch = D + 4;  // floats per row of a wave's partial
  constexpr int kVBytes = W * kStages * kTileBytes;
  constexpr int kPartBytes = W * kRows * kPitch * 4;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kVBytes > kPartBytes ? kVBytes : kPartBytes];
  __shared__ float msm[W][kRows], lsm[W][kRows];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int slot = blockIdx.x / a.units;
  const int unit = blockIdx.x - slot * a.units;
  const int hk = unit % a.Hkv;
  const int rb = unit / a.Hkv;
  Share s;
  if (!share_of(a, slot, s)) return;  // the whole workgroup

  const uint16_t* kbase = static_cast<const uint16_t*>(a.k) + s.b * a.seq + hk * a.head;
  const uint16_t* vbase = static_cast<const uint16_t*>(a.v) + s.b * a.seq + hk * a.head;
  const int kb0 = s.k0 + wave * TK;
  const int ntiles = s.k1 > kb0 ? (s.k1 - kb0 + W * TK - 1) / (W * TK) : 0;

  VTile<D> ld;
  ld.init(a.row, lane);
  const uint32_t vlds = t128::lds_addr(smem) + wave * kStages * kTileBytes;
  const uint8_t* vmem = smem + wave * kStages * kTileBytes;
  auto issue = [&](int j) {  // V tile j into stage j % kStages
    ld.template load<NT>(vbase, a.row, kb0 + j * (W * TK), s.k1, vlds + (j % kStages) * kTileBytes, lane,
                          &kZeroRow);
  };
  auto kload = [&](int j, bf16x8 (&kr)[MB][KS]) {  // lane (c, g): key 16 mb + c, dims 32 kk + 8 g
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const int row = min(kb0 + j * (W * TK) + 16 * mb + c, s.k1 - 1);
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        const bf16x8* at = reinterpret_cast<const bf16x8*>(kbase + row * a.row + 32 * kk + 8 * g);
        kr[mb][kk] = NT ? __builtin_nontemporal_load(at) : *at;
      }
    }
  };

  bf16x8 kra[MB][KS], krb[MB][KS];
  if (ntiles > 0) {
    issue(0);
    kload(0, kra);
  }
  bf16x8 qreg[NB][KS];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = rb * kRows + 16 * nb + c, rr = r < a.R ? r : 0;
    const int64_t qi = ((int64_t)s.b * a.N + rr / a.group) * a.Hq + hk * a.group + rr % a.group;
    const uint16_t* qrow = static_cast<const uint16_t*>(a.q) + qi * D;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      qreg[nb][kk] = *reinterpret_cast<const bf16x8*>(qrow + 32 * kk + 8 * g);
      if (r >= a.R) qreg[nb][kk] = bf16x8{};
    }
  }
  t128::wait_vmem();  // Q is there (the compiler cannot count the tile loads below)

  int voff[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) voff[db] = VTile<D>::tr_off(16 * db, lane);
  f32x4 o[NB][DB];
  float mrow[NB], lsum[NB];  // running maximum (log2 units), lane-partial sum of p
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int db = 0; db < DB; ++db) o[nb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    mrow[nb] = -INFINITY;
    lsum[nb] = 0.f;
  }

  // Tile j: wait for V(j) and K(j) (issued at tile j - 1), issue V(j + 1) into
  // the stage that tile j - 1 is done with and K(j + 1) into the other
  // registers, then compute.
  auto tile = [&](int j, bf16x8 (&kc)[MB][KS], bf16x8 (&kn)[MB][KS]) {
    t128::wait_vmem();
    if (j + 1 < ntiles) {
      issue(j + 1);
      if constexpr (NB < 4) kload(j + 1, kn);
    }
    const uint8_t* vt = vmem + (j % kStages) * kTileBytes;
    const int left = s.k1 - (kb0 + j * (W * TK));  // keys of the split from this tile on
    f32x4 sc[NB][MB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) sc[nb][mb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < KS; ++kk)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) sc[nb][mb] = mfma16x16x32(kc[mb][kk], qreg[nb][kk], sc[nb][mb]);
    if constexpr (NB == 4) {
      __builtin_amdgcn_sched_barrier(0);
      if (j + 1 < ntiles) kload(j + 1, kc);
    }
    if (left < TK) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * mb + i >= left - 4 * g) sc[nb][mb][i] = -INFINITY;
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float mx = -INFINITY;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
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
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = fast_exp2(fmaf(sc[nb][mb][i], a.sl2, -muse));
          lsum[nb] += p;
          sc[nb][mb][i] = p;
        }
    }
#pragma unroll
    for (int k2 = 0; k2 < TK / 32; ++k2) {
      bf16x8 pb[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) pb[nb] = pack_bf16x8(sc[nb][2 * k2], sc[nb][2 * k2 + 1]);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const uint8_t* p = vt + voff[db] + 32 * k2 * 2 * D;
        const bf16x8 va = concat_bf16x4(t128::ds_read_tr(p), t128::ds_read_tr(p + 16 * 2 * D));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) o[nb][db] = mfma16x16x32(va, pb[nb], o[nb][db]);
      }
    }
  };
  if constexpr (NB == 4) {
    for (int j = 0; j < ntiles; ++j) tile(j, kra, kra);
  } else {
    for (int j = 0; j < ntiles; j += 2) {
      tile(j, kra, krb);
      if (j + 1 < ntiles) tile(j + 1, krb, kra);
    }
  }

  auto emit = [&](int r, int d, const f32x4& acc, float L, float M) {
    const int64_t pr = partial_row(a, r, hk, slot);
    *reinterpret_cast<f32x4*>(a.po + pr * D + d) = acc;
    if (d == 0) a.ps[pr] = make_float2(M, L);
  };
  // The waves' partials, brought to each row's maximum, meet in LDS.
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
    if (g == 0) msm[wave][16 * nb + c] = mrow[nb];
  __syncthreads();  // also: every wave is done with its V tiles
  float* part = reinterpret_cast<float*>(smem);
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
      *reinterpret_cast<f32x4*>(part + (wave * kRows + 16 * nb + c) * kPitch + 16 * db + 4 * g) = o[nb][db] * f;
  }
  __syncthreads();
  constexpr int kPer = D / 4;  // threads per row
  for (int it = threadIdx.x; it < kRows * kPer; it += 64 * W) {
    const int rr = it / kPer, d = 4 * (it % kPer);
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
    emit(r, d, acc, L, M);
  }
}

// ---------------------------------- the past, bf16, head_dim 128, many rows --

// Many query rows: the matrix cores and the softmax beside them bound it.  Eight
// waves of 32 rows over 64-key tiles of K and V in LDS (tile128.h), filled by LDS
// DMA; S^T = K Q^T and O^T += V^T P^T on 32 x 32 x 16 products.  Iteration j issues
// the products of S^T for tile j + 1 and beside them, on the VALU, the softmax of
// tile j, then O^T += V_j^T P_j^T; K runs one tile ahead of V, two buffers each,
// one barrier per tile.
//   RW = 8: 256 rows that share every tile.
//   RW = 4: 128 rows; waves 0-3 take the even tiles, 4-7 the odd ones (buffers of
//           their own), and the halves meet in LDS: two waves a SIMD, which the
//           products need to hide their LDS reads (32 tokens of 32/8 heads over
//           262,000 keys 209 us with the merge; with four waves 12 to 20 more).
// 256 rows take 317 us there (64 tokens, 867 TFLOP/s, with the merge): the softmax
// of a tile does not hide behind the products entirely.
// Probabilities go to the products in bf16 (their sum stays fp32), relative to the
// row's exact running maximum, so the largest so far is not rounded: a relative
// error of 1.73e-3 at 26 tokens over 16,000 keys, 1.64e-3 of it the output's own
// rounding.  A reference that is raised by factors of 2^8 only saves most of the
// rescaling (64 tokens over 262,000 keys, in all, 306 us against 317; over 16,000 62
// against 59), but rounds the largest too: 2.09e-3.
template <int RW, bool NT>
__global__ __launch_bounds__(512, 1) void cache_tile128_kernel(AttnArgs a) {
  constexpr int D = 128, BN = 64, KG = 8 / RW;
  constexpr int kTileB = BN * t128::kRowBytes;
  constexpr int kPitch = D + 4;
  constexpr int kBufs = 4 * KG * kTileB, kPart = KG > 1 ? 32 * RW * kPitch * 4 : 0;
  static_assert(kPart <= kBufs, "the halves meet in the tiles' buffers");
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kBufs];
  __shared__ float2 stat_s[32 * RW];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = KG > 1 ? wave >> 2 : 0;  // which tiles
  const int rw = KG > 1 ? wave & 3 : wave;
  const int kc = lane & 31;  // this lane's row within the wave
  const int hh = lane >> 5;  // which half of each 8-key group the lane holds
  const int slot = blockIdx.x / a.units;
  const int unit = blockIdx.x - slot * a.units;
  const int hk = unit % a.Hkv;
  const int rb = unit / a.Hkv;
  Share s;
  if (!share_of(a, slot, s)) return;  // the whole workgroup

  const uint16_t* kbase = static_cast<const uint16_t*>(a.k) + s.b * a.seq + hk * a.head;
  const uint16_t* vbase = static_cast<const uint16_t*>(a.v) + s.b * a.seq + hk * a.head;
  // In a vector register: as a scalar it makes the compiler merge the loop's
  // branches, at the price of 336 to 420 bytes of scratch a lane.
  const int all = opaque((s.k1 - s.k0 + BN - 1) / BN);
  const int steps = (all + KG - 1) / KG;                 // tiles of the longer half
  const int ntiles = KG > 1 ? (all - kg + 1) / 2 : all;  // of this wave's
  const int r = 32 * (rb * RW + rw) + kc;

  t128::RowLoader<BN, RW> ld;
  ld.init(a.row, rw, lane);
  const uint32_t lds0 = t128::lds_addr(smem) + kg * 4 * kTileB;
  const uint8_t* const kbuf = smem + kg * 4 * kTileB;
  const uint8_t* const vbuf = kbuf + 2 * kTileB;
  // Tile j of K (what = 0) or V (1), if there is one, into buffer buf.
  auto issue = [&](int what, int j, int buf) {
    if (j < ntiles)
      ld.template load<false, NT>(what ? vbase : kbase, a.row, s.k0 + (KG * j + kg) * BN, s.k1,
                                  lds0 + (2 * what + buf) * kTileB, rw, lane, &kZeroRow);
  };
  issue(0, 0, 0);
  issue(1, 0, 0);
  issue(0, 1, 1);

  bf16x8 qreg[D / 16];  // lane: row r, dims 16 t + 8 hh .. + 7
  {
    const int rr = r < a.R ? r : 0;
    const int64_t qi = ((int64_t)s.b * a.N + rr / a.group) * a.Hq + hk * a.group + rr % a.group;
    const uint16_t* qrow = static_cast<const uint16_t*>(a.q) + qi * D;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) qreg[t] = *reinterpret_cast<const bf16x8*>(qrow + 16 * t + 8 * hh);
  }
  const int roff0 = t128::row_chunk_off(kc, hh);
  const int toff0 = t128::tr32_off(0, lane), toff1 = t128::tr32_off(1, lane);
  int koff[8], voff0[4], voff1[4];
#pragma unroll
  for (int t = 0; t < 8; ++t) koff[t] = opaque(roff0 ^ (32 * t));
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    voff0[u] = opaque(toff0 ^ (64 * u));
    voff1[u] = opaque(toff1 ^ (64 * u));
  }
  f32x16 o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = f32x16{};
  float mrun = -INFINITY;                     // log2 units, shared by the lanes l, l ^ 32
  float lsum = 0.f;                           // lane-partial, relative to mrun

  auto kread = [&](const uint8_t* kt, int i) {  // S step i: t = i / 2, mb = i % 2
    return *reinterpret_cast<const bf16x8*>(kt + koff[i >> 1] + (i & 1) * 32 * t128::kRowBytes);
  };
  auto vread = [&](const uint8_t* vt, int i) {  // PV step i: u = i / 4, dims 32 (i % 4) ..
    const int o0 = voff0[i & 3] + (i >> 2) * 16 * t128::kRowBytes;
    const int o1 = voff1[i & 3] + (i >> 2) * 16 * t128::kRowBytes;
    return concat_bf16x4(t128::ds_read_tr(vt + o0), t128::ds_read_tr(vt + o1));
  };
  auto scores_only = [&](const uint8_t* kt, f32x16 (&x)[2]) {
    bf16x8 A[2] = {kread(kt, 0), kread(kt, 1)};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i & 1] = mfma32x32x16(A[i & 1], qreg[i >> 1], i < 2 ? f32x16{} : x[i & 1]);
      if (i + 2 < 16) A[i & 1] = kread(kt, i + 2);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // left: keys of the split from this tile on (read on its last tile alone).
  auto iteration = [&](auto last_tag, const uint8_t* kt, const uint8_t* vt, f32x16 (&sc)[2],
                       f32x16 (&sn)[2], int left) {
    constexpr bool LAST = decltype(last_tag)::value;
    bf16x8 A[2], B[2], pb[4];
    if constexpr (!LAST) {
      A[0] = kread(kt, 0);
      A[1] = kread(kt, 1);
    }
    const int klim = left - 4 * hh;
    float pmax = -INFINITY, muse = 0.f;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if constexpr (!LAST) {
        sn[i & 1] = mfma32x32x16(A[i & 1], qreg[i >> 1], i < 2 ? f32x16{} : sn[i & 1]);
        if (i + 2 < 16) A[i & 1] = kread(kt, i + 2);
      }
      if (i < 4) {  // the maximum, 8 scores per step
#pragma unroll
        for (int e = 8 * i; e < 8 * i + 8; ++e) {
          const int mb = e >> 4, v = e & 15;
          if constexpr (LAST)
            if (32 * mb + 8 * (v >> 2) + (v & 3) >= klim) sc[mb][v] = -INFINITY;
          pmax = fmaxf(pmax, sc[mb][v]);
        }
      }
      if (i == 7) {
        const float mx = xor32_max(pmax) * a.sl2;
        if (__any(mx > mrun)) {
          const float alpha = mx > mrun ? fast_exp2(mrun - mx) : 1.f;  // mrun = -inf: 0
          mrun = fmaxf(mrun, mx);
          lsum *= alpha;
#pragma unroll
          for (int d = 0; d < 4; ++d) o[d] *= alpha;
        }
        muse = mrun == -INFINITY ? 0.f : mrun;
      }
      if (i >= 8) {  // probabilities, 4 per step
#pragma unroll
        for (int e = 4 * (i - 8); e < 4 * (i - 8) + 4; ++e) {
          const int mb = e >> 4, v = e & 15;
          const float p = fast_exp2(fmaf(sc[mb][v], a.sl2, -muse));
          lsum += p;
          sc[mb][v] = p;
        }
      }
      if (i == 11 || i == 15) {  // B operands of keys 32 mb .. 32 mb + 31
        const int mb = (i - 11) >> 2;
#pragma unroll
        for (int u2 = 0; u2 < 2; ++u2) {
          const int e0 = 8 * u2;
          pb[2 * mb + u2] = pack_bf16x8(
              f32x4{sc[mb][e0], sc[mb][e0 + 2], sc[mb][e0 + 4], sc[mb][e0 + 6]},
              f32x4{sc[mb][e0 + 1], sc[mb][e0 + 3], sc[mb][e0 + 5], sc[mb][e0 + 7]});
        }
      }
      if (i == 14) B[0] = vread(vt, 0);
      if (i == 15) B[1] = vread(vt, 1);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      o[i & 3] = mfma32x32x16(B[i & 1], pb[i >> 2], o[i & 3]);
      if (i + 2 < 16) B[i & 1] = vread(vt, i + 2);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto stage = [&](int j, auto parity, f32x16 (&sc)[2], f32x16 (&sn)[2]) {
    constexpr int P = decltype(parity)::value;  // j % 2
    t128::wait_vmem();
    __syncthreads();
    issue(0, j + 2, P);
    issue(1, j + 1, P ^ 1);
    if (j + 1 < ntiles)
      iteration(std::false_type{}, kbuf + (P ^ 1) * kTileB, vbuf + P * kTileB, sc, sn, BN);
    else if (j < ntiles)
      iteration(std::true_type{}, kbuf, vbuf + P * kTileB, sc, sn, s.k1 - s.k0 - (KG * j + kg) * BN);
  };
  f32x16 sa[2], sb[2];
  t128::wait_vmem();
  __syncthreads();
  if (ntiles > 0) scores_only(kbuf, sa);
  for (int j = 0; j < steps; j += 2) {
    stage(j, std::integral_constant<int, 0>{}, sa, sb);
    if (j + 1 < steps) stage(j + 1, std::integral_constant<int, 1>{}, sb, sa);
  }

  float f = 1.f, lt = xor32_sum(lsum);
  float* part = reinterpret_cast<float*>(smem) + (32 * rw + kc) * kPitch + 4 * hh;
  float wb = 0.f;
  if constexpr (KG > 1) {  // the odd tiles' half hands over
    __syncthreads();  // the tiles are done with
    if (kg == 1) {
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int w = 0; w < 4; ++w)
          *reinterpret_cast<f32x4*>(part + 32 * d + 8 * w) =
              f32x4{o[d][4 * w], o[d][4 * w + 1], o[d][4 * w + 2], o[d][4 * w + 3]};
      if (hh == 0) stat_s[32 * rw + kc] = make_float2(mrun, lt);
    }
    __syncthreads();
    if (kg == 1) return;
    const float2 st = stat_s[32 * rw + kc];
    const float top = fmaxf(mrun, st.x);
    const float wa = mrun == -INFINITY ? 0.f : fast_exp2(mrun - top);
    wb = st.x == -INFINITY ? 0.f : fast_exp2(st.x - top);
    f *= wa;
    lt = lt * wa + st.y * wb;
    mrun = top;
  }
  if (r < a.R) {
    const int64_t pr = partial_row(a, r, hk, slot);
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        f32x4 x = f32x4{o[d][4 * w], o[d][4 * w + 1], o[d][4 * w + 2], o[d][4 * w + 3]} * f;
        if constexpr (KG > 1) x += *reinterpret_cast<const f32x4*>(part + 32 * d + 8 * w) * wb;
        *reinterpret_cast<f32x4*>(a.po + pr * D + 32 * d + 8 * w + 4 * hh) = x;
      }
    if (hh == 0) a.ps[pr] = make_float2(mrun, lt);
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

// WPR waves (a workgroup) per query row share its splits and the keys of its
// chain and meet in LDS.  Lane 16 u + j holds 4-element chunks j, j + 16, .. of
// the head dim (NI of them) for the u-th of every four keys (splits) of the
// wave.  A row costs few bytes and would cost many memory latencies, so what
// does not depend on the chain (the first partials) is read before the chain
// is followed, and the keys and values of kKeys steps together (64 tokens of 32
// heads over 32 splits, chains of some ten keys: 16.7 us, 17.5 with one step at
// a time).
template <typename T, int NI, int WPR>
__global__ __launch_bounds__(64 * WPR) void cache_merge_kernel(AttnArgs a) {
  constexpr int kStep = 4 * WPR;                              // splits and keys of a step
  constexpr int kFirst = (WPR == 1 ? 8 : 4) / (NI > 1 ? NI : 2);  // steps of partials read up front
  constexpr int kKeys = WPR == 1 && NI < 4 ? 4 : 1;               // steps of keys read together
  __shared__ uint16_t chain_s[WPR][kCacheMaxTokens];
  __shared__ float top_s[WPR], l_s[WPR];
  __shared__ f32x4 acc_s[WPR][16 * NI];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = lane & 15, u = lane >> 4;
  const int row = blockIdx.x;
  const int h = row % a.Hq;
  const int bi = row / a.Hq;
  const int i = bi % a.N, b = bi / a.N;
  const int hk = h / a.group;
  const int past = a.past[b];
  const int nch = a.D / 4;

  // The parents of the tokens up to this one, over the lanes.
  int par[kCacheMaxTokens / 64];
#pragma unroll
  for (int x = 0; x < kCacheMaxTokens / 64; ++x) {
    const int at = 64 * x + lane;
    par[x] = at - 1;
    if (a.parents != nullptr && 64 * x <= i) par[x] = a.parents[(int64_t)b * a.N + min(at, a.N - 1)];
  }
  f32x4 qv[NI];
  const T* qp = static_cast<const T*>(a.q) + (int64_t)row * a.D;
#pragma unroll
  for (int x = 0; x < NI; ++x) qv[x] = load_w<T, 4>(qp, 4 * (j + 16 * x), a.D, true);

  const int2 deal = a.deal[b];
  const int splits = deal.y;
  const int64_t pr0 = ((int64_t)i * a.Hq + h) * a.slots + deal.x;
  f32x4 po[kFirst][NI];
  float2 ps[kFirst];
#pragma unroll
  for (int f = 0; f < kFirst; ++f) {
    const int s = kStep * f + 4 * wave + u;
    const int64_t pr = pr0 + min(s, splits - 1);
    ps[f] = a.ps[pr];
#pragma unroll
    for (int x = 0; x < NI; ++x) po[f][x] = load_w<float, 4>(a.po + pr * a.D, 4 * (j + 16 * x), a.D, true);
  }

  // The chain of parents, the token itself first.
  uint16_t* chain = chain_s[wave];
  bool there = past >= 0 && past < a.C && i < a.C - past;
  int n = 0;
  for (int at = i; there;) {  // at falls with every step
    if (lane == 0) chain[n] = (uint16_t)at;
    ++n;
    int p = -2;
#pragma unroll
    for (int x = 0; x < kCacheMaxTokens / 64; ++x)
      if (at >> 6 == x) p = __builtin_amdgcn_readlane(par[x], at & 63);
    if (p == -1) break;
    there = p >= 0 && p < at;
    at = p;
  }
  const int64_t si = ((int64_t)b * a.Hq + h) * a.N + i;
  T* out = static_cast<T*>(a.out) + (int64_t)row * a.D;
  if (!there) {  // the whole workgroup
    if (wave == 0) {
#pragma unroll
      for (int x = 0; x < NI; ++x)
        if (u == 0 && j + 16 * x < nch) store_vec4<T>(out + 4 * (j + 16 * x), f32x4{0.f, 0.f, 0.f, 0.f});
      if (lane == 0) {
        if (a.m) a.m[si] = -INFINITY;
        if (a.l) a.l[si] = 0.f;
      }
    }
    return;
  }
  wave_lds_sync();

  // The chain's keys: every group of 16 lanes has a running maximum of its own.
  const T* kb = static_cast<const T*>(a.k) + b * a.seq + hk * a.head + past * a.row;
  const T* vb = static_cast<const T*>(a.v) + b * a.seq + hk * a.head + past * a.row;
  f32x4 acc[NI];
#pragma unroll
  for (int x = 0; x < NI; ++x) acc[x] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  for (int x0 = 4 * wave + u; x0 < n; x0 += kKeys * kStep) {
    f32x4 kx[kKeys][NI], vx[kKeys][NI];
#pragma unroll
    for (int f = 0; f < kKeys; ++f) {
      const int64_t off = chain[min(x0 + kStep * f, n - 1)] * a.row;
#pragma unroll
      for (int y = 0; y < NI; ++y) {
        kx[f][y] = load_w<T, 4>(kb + off, 4 * (j + 16 * y), a.D, true);
        vx[f][y] = load_w<T, 4>(vb + off, 4 * (j + 16 * y), a.D, true);
      }
    }
    float s[kKeys], mnew = m;
#pragma unroll
    for (int f = 0; f < kKeys; ++f) {
      f32x4 s4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int y = 0; y < NI; ++y) s4 += qv[y] * kx[f][y];
      s[f] = (s4[0] + s4[1]) + (s4[2] + s4[3]);
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1)
#pragma unroll
      for (int f = 0; f < kKeys; ++f) s[f] += __shfl_xor(s[f], o, 64);
#pragma unroll
    for (int f = 0; f < kKeys; ++f) {
      s[f] *= a.sl2;
      if (x0 + kStep * f < n) mnew = fmaxf(mnew, s[f]);
    }
    const float muse = mnew == -INFINITY ? 0.f : mnew;
    const float alpha = exp2f(m - muse);  // m = -inf: 0
    l *= alpha;
#pragma unroll
    for (int y = 0; y < NI; ++y) acc[y] *= alpha;
    m = mnew;
#pragma unroll
    for (int f = 0; f < kKeys; ++f) {
      if (x0 + kStep * f >= n) continue;
      const float p = exp2f(s[f] - muse);
      l += p;
#pragma unroll
      for (int y = 0; y < NI; ++y) acc[y] += vx[f][y] * p;
    }
  }

  // The row's maximum, and everything relative to it.
  float top = m;
#pragma unroll
  for (int f = 0; f < kFirst; ++f) top = fmaxf(top, ps[f].x);  // (a re-read split changes nothing)
  for (int s = kStep * kFirst + 64 * wave + lane; s < splits; s += 64 * WPR)
    top = fmaxf(top, a.ps[pr0 + s].x);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if constexpr (WPR > 1) {
    if (lane == 0) top_s[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WPR; ++w) top = fmaxf(top, top_s[w]);
  }
  const float muse = top == -INFINITY ? 0.f : top;
  {
    const float alpha = exp2f(m - muse);
    l *= alpha;
#pragma unroll
    for (int x = 0; x < NI; ++x) acc[x] *= alpha;
  }
#pragma unroll
  for (int f = 0; f < kFirst; ++f) {
    if (kStep * f + 4 * wave + u >= splits) continue;
    const float w = exp2f(ps[f].x - muse);  // a split without keys: 0
    l += w * ps[f].y;
#pragma unroll
    for (int x = 0; x < NI; ++x) acc[x] += po[f][x] * w;
  }
#pragma unroll(NI == 4 ? 1 : 4)
  for (int s = kStep * kFirst + 4 * wave + u; s < splits; s += kStep) {
    const int64_t pr = pr0 + s;
    const float2 st = a.ps[pr];
    const float w = exp2f(st.x - muse);
    l += w * st.y;
#pragma unroll
    for (int x = 0; x < NI; ++x)
      acc[x] += load_w<float, 4>(a.po + pr * a.D, 4 * (j + 16 * x), a.D, true) * w;
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
    l = l_s[0];
#pragma unroll
    for (int x = 0; x < NI; ++x) acc[x] = acc_s[0][j + 16 * x];
#pragma unroll 4
    for (int w = 1; w < WPR; ++w) {
      l += l_s[w];
#pragma unroll
      for (int x = 0; x < NI; ++x) acc[x] += acc_s[w][j + 16 * x];
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int x = 0; x < NI; ++x)
    if (u == 0 && j + 16 * x < nch) store_vec4<T>(out + 4 * (j + 16 * x), acc[x] * inv);
  if (lane == 0) {
    if (a.m) a.m[si] = top == -INFINITY ? top : top * kLn2;
    if (a.l) a.l[si] = l;
  }
}

// ------------------------------------------------------------------- host --

// Query rows from which a wave each is enough for the chip: more waves a row cost
// more instructions than they save latency (32 heads: 64 tokens 16.7 us against
// 18.4 with four, 26 tokens 9.8 against 8.8).
constexpr int64_t kManyRows = 1024;

// Workgroups for a whole chip, one a CU: each split costs a partial that is
// written and merged.  The fp32 form takes two where it waits for its products
// and has the registers for them: 64 tokens of 32/8 heads over 16,000 keys, in
// all, 129 us against 164 at head_dim 64 and 242 against 274 at 128, but 8 tokens
// of 128 48 against 45, one 40 against 29.
constexpr int64_t kWanted = 256;

// Bytes of K and V, at their capacity, that all row blocks of 32 read together,
// up to which those are the best form for more rows too: the second block finds
// in the caches what the first has read, and the waves need not wait for each
// other.  Beyond, 64, 128 or 256 rows a workgroup read less.  32/8 heads of 128,
// in all: 16 tokens 18.9 us against 21.8 at 4,000 keys, 30.2 against 33.6 at
// 24,000, 70 against 58 at 60,000; 26 tokens 21.0 against 25.1 at 4,000, 35.3
// against 33.2 at 16,000; 64 tokens 21.6 against 28.3 at 500, 30.4 against 40.8 at
// 4,000, 59 against 53 at 16,000.  (The capacity decides: 64 tokens over 500 keys
// take 31 us in a cache of 564 rows, 35 in a larger one, 26 over 4,000 23 and 27.)
// Of 64: 16 tokens 26.2 against 28.0 at 60,000
// keys, 148 against 104 at 262,000; 26 tokens 16.5 against 18.6 at 4,000, 50.7
// against 43.0 at 60,000.
constexpr int64_t kBlockBytes = 240 << 20;

enum class Form { kFp32, kStream, kTiled };

struct Plan {
  Form form;
  int waves;  // of a workgroup
  int rows;   // of a workgroup (fp32: 16 for each of its row blocks)
  int units, slots;
};

Plan make_plan(const CacheProblem& p) {
  const int64_t R = (int64_t)p.N * (p.Hq / p.Hkv);
  const int64_t tiles = (int64_t)p.B * ((p.C + kTile - 1) / kTile);
  const bool bf16 = p.dtype == 1 && !p.precise && (p.D == 64 || p.D == 128);
  const bool blocks = R <= 32 || (R + 31) / 32 * p.B * p.C * p.Hkv * p.D * 4 <= kBlockBytes;
  Plan x;
  x.waves = 4;
  if (!bf16) {
    x.form = Form::kFp32;
    x.rows = R <= 16 ? 16 : R <= 32 ? 32 : 64;
  } else if (blocks || p.D == 64) {
    x.form = Form::kStream;
    x.rows = R <= 16 ? 16 : blocks ? 32 : 64;
  } else {
    x.form = Form::kTiled;
    x.waves = 8;
    x.rows = R <= 128 ? 128 : 256;
  }
  x.units = (int)((R + x.rows - 1) / x.rows * p.Hkv);
  const bool twice = x.form == Form::kFp32 && (p.D <= 96 || R > 64);
  const int64_t want = twice ? 2 * kWanted : kWanted;
  const int64_t slots = std::max<int64_t>(1, std::min<int64_t>(want / x.units, tiles));
  // A batch of nearly as many sequences as slots, or more, has some left for its
  // long ones: 39 sequences of 300 keys and one of 16,000 take 59 us, with a slot
  // each 292.
  x.slots = (int)(p.B > kTightBatch ? slots + p.B : std::max<int64_t>(slots, p.B > 1 ? p.B + slots / 2 : 1));
  return x;
}

}  // namespace

size_t cache_attn_bytes(const CacheProblem& p) {
  const Plan x = make_plan(p);
  return (size_t)x.slots * p.N * p.Hq * (p.D + 2) * sizeof(float) + (size_t)p.B * sizeof(int2);
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
  a.ps = reinterpret_cast<float2*>(a.po + prows * p.D);
  a.deal = reinterpret_cast<int2*>(a.ps + prows);
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
  a.wave_rows = x.rows / 16;
  a.seq = p.seq;
  a.row = p.row;
  a.head = p.head;
  a.sl2 = p.sl2;
  auto prefix = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(x.slots * x.units)), dim3(64 * x.waves), 0, st, a);
  };
  auto fp32 = [&](auto t) {
    using T = decltype(t);
    if (p.D <= 16) prefix(cache_prefix32_kernel<T, 1>);
    else if (p.D <= 32) prefix(cache_prefix32_kernel<T, 2>);
    else if (p.D <= 64) prefix(cache_prefix32_kernel<T, 4>);
    else if (p.D <= 96) prefix(cache_prefix32_kernel<T, 6>);
    else if (p.D <= 128) prefix(cache_prefix32_kernel<T, 8>);
    else prefix(cache_prefix32_kernel<T, 16>);
  };
  const bool once = x.units == p.Hkv;  // the cache is read once: L2 need not keep it
  auto stream = [&](auto d) {
    constexpr int kD = decltype(d)::value;
    constexpr bool kNt = kD == 128;
    if (x.rows == 16) prefix(cache_stream_kernel<kD, 1, kNt>);
    else if (x.rows == 32 && once) prefix(cache_stream_kernel<kD, 2, kNt>);
    else if (x.rows == 32) prefix(cache_stream_kernel<kD, 2, false>);
    else if constexpr (kD == 64) prefix(cache_stream_kernel<kD, 4, false>);
  };
  if (x.form == Form::kFp32) {
    if (p.dtype == 1) fp32(uint16_t{});
    else fp32(float{});
  } else if (x.form == Form::kStream) {
    if (p.D == 64) stream(std::integral_constant<int, 64>{});
    else stream(std::integral_constant<int, 128>{});
  } else {
    if (x.rows == 128) prefix(cache_tile128_kernel<4, true>);
    else if (once) prefix(cache_tile128_kernel<8, true>);
    else prefix(cache_tile128_kernel<8, false>);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t rows = (int64_t)p.B * p.N * p.Hq;
  auto merge = [&](auto kernel, int waves) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(64 * waves), 0, st, a);
  };
  auto merge_dim = [&](auto t, auto ni) {
    using T = decltype(t);
    constexpr int kNI = decltype(ni)::value;
    if (rows < kManyRows) merge(cache_merge_kernel<T, kNI, 4>, 4);
    else merge(cache_merge_kernel<T, kNI, 1>, 1);
  };
  auto merge_type = [&](auto t) {
    if (p.D <= 64) merge_dim(t, std::integral_constant<int, 1>{});
    else if (p.D <= 128) merge_dim(t, std::integral_constant<int, 2>{});
    else merge_dim(t, std::integral_constant<int, 4>{});
  };
  if (p.dtype == 1) merge_type(uint16_t{});
  else merge_type(float{});
  return hipGetLastError();
}

}  // namespace lc
