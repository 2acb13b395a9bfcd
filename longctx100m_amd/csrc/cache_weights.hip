// Accumulated attention weight of the rows of a KV cache (gfx950): with the
// statistics of the attention given,
//   w[h][j] = sum over the query rows r of KV head h that see row j of
//             exp(s_rj - m_r) / l_r = sum exp2(s'_rj - lse2_r),
// s' in log2 units and lse2 = m log2(e) + log2(l), so that a row costs one
// subtraction and one exp2 per key.  The price is lse2's own rounding in the
// exponent, 2^-24 of its value at most: 1.0e-7 from 64 bits for 512 tokens behind
// 32,000 keys (m and l taken apart: 5e-8), 4.6e-7 for one token over 262,000 (4.1e-7).
// Keys are stationary and the query rows
// stream past them, which makes the sum over rows a sum within a lane: no
// atomics, a fixed order.  Rows that a key is not seen by are left out by
// selection, not by a factor, so a NaN in an unseen place stays there.
#include "common.h"
#include "cache.h"
#include "kernels.h"
#include "tile128.h"
#include "tile32.h"

#include <algorithm>
#include <type_traits>

namespace lc {
namespace {

struct WeightArgs {
  const void *q, *k;
  const float *m, *l, *w;
  float* w_out;
  const int32_t *past, *parents;
  int B, N, C, Hq, Hkv, D, group, R;
  int kblocks;  // workgroups of a KV head
  int64_t seq, row, head;
  float sl2;
};

// Which new tokens each new token sees, one bit each (a token that is not there: none).
constexpr int kWords = kCacheMaxTokens / 32;
struct Tree {
  uint32_t seen[kCacheMaxTokens][kWords];
  int parent[kCacheMaxTokens];
};

// By a workgroup of 256 threads; ends with a barrier.
__device__ __forceinline__ void build_tree(Tree& t, const int32_t* parents, int N) {
  const int i = threadIdx.x;
  t.parent[i] = i < N ? parents[i] : -2;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < kWords; ++x) t.seen[i][x] = 0;
  int at = i;
  bool there = i < N;
  while (there) {  // at falls with every step
    t.seen[i][at >> 5] |= 1u << (at & 31);
    const int p = t.parent[at];
    if (p == -1) break;
    there = p >= 0 && p < at;
    at = p;
  }
  if (!there) {
#pragma unroll
    for (int x = 0; x < kWords; ++x) t.seen[i][x] = 0;
  }
  __syncthreads();
}

// A row's log-sum-exp in log2 units, and whether the row gives anything.
__device__ __forceinline__ float row_lse(float m, float l) {
  return fmaf(m, kLog2e, log2f(l));
}
__device__ __forceinline__ bool gives(float m, float l) { return l > 0.f && m != -INFINITY; }

// fp32 products, any head_dim: a wave holds 16 keys, and the query rows of its KV
// head, (token, head of the group) by token, pass by in tiles of 16 that the
// four waves read together: fragments in LDS, each lane at its own 16 bytes,
// with the rows' statistics, two buffers, the next tile's loads in flight over a
// tile.  32/8 heads of 128 over 16,000 keys: 64 tokens 107 us (80 TFLOP/s), 8 tokens
// 23, one 16 (4.1 TB/s); with each wave reading the rows for itself 180, 34 and 20.
template <typename T, int NJ>
__global__ __launch_bounds__(256) void cache_weights32_kernel(WeightArgs a) {
  constexpr int kF = (NJ + 3) / 4;  // fragments that a wave reads
  __shared__ Tree tree;
  __shared__ __attribute__((aligned(16))) f32x4 q_s[2][NJ * 64];
  __shared__ __attribute__((aligned(16))) float lse_s[2][16];
  __shared__ __attribute__((aligned(16))) int tok_s[2][16];  // -1: a row that gives nothing
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int kblk = blockIdx.x % a.kblocks;
  const int bh = blockIdx.x / a.kblocks;
  const int hk = bh % a.Hkv, b = bh / a.Hkv;
  const int past_in = a.past[b];
  const int past = min(past_in, a.C);
  const int len = (int)min((int64_t)past + a.N, (int64_t)a.C);
  if (past_in < 0 || 64 * kblk >= len) return;  // the whole workgroup
  const int there = len - past;  // tokens whose row lies in the cache

  const T* qb = static_cast<const T*>(a.q) + ((int64_t)b * a.N * a.Hq + (int64_t)hk * a.group) * a.D;
  const int64_t sb = ((int64_t)b * a.Hq + hk * a.group) * a.N;
  f32x4 qn[kF];
  float mn = 0.f, ln = 0.f;
  auto fetch = [&](int t) {
    {
      const int r = 16 * t + c, rr = r < a.R ? r : 0;
      const T* qp = qb + ((int64_t)(rr / a.group) * a.Hq + rr % a.group) * a.D;
#pragma unroll
      for (int f = 0; f < kF; ++f) {
        const int j = wave + 4 * f;
        qn[f] = load_w<T, 4>(qp, r < a.R ? 16 * j + 4 * g : a.D, a.D, true);
      }
    }
    if (threadIdx.x < 16) {
      const int r = 16 * t + (int)threadIdx.x, rr = r < a.R ? r : 0;
      const int64_t si = sb + (int64_t)(rr % a.group) * a.N + rr / a.group;
      mn = a.m[si];
      ln = a.l[si];
    }
  };
  auto put = [&](int t, int buf) {
#pragma unroll
    for (int f = 0; f < kF; ++f) {
      const int j = wave + 4 * f;
      if (j < NJ) q_s[buf][64 * j + lane] = qn[f];
    }
    if (threadIdx.x < 16) {
      const int r = 16 * t + (int)threadIdx.x, token = r / a.group;
      const bool ok = r < a.R && token < there && gives(mn, ln);
      lse_s[buf][threadIdx.x] = ok ? row_lse(mn, ln) : 0.f;
      tok_s[buf][threadIdx.x] = ok ? token : -1;
    }
  };
  // A chain's rows before the first token that sees one of the keys see none.
  const int first = a.parents ? 0 : max(0, 64 * kblk - past) * a.group / 16;
  const bool any = 16 * first < a.R;
  if (any) fetch(first);

  const int key0 = 64 * kblk + 16 * wave;
  const int key = key0 + c;
  const int nkey = key - past;  // the token whose row this is, if >= 0
  const T* kb = static_cast<const T*>(a.k) + b * a.seq + hk * a.head;
  f32x4 kr[NJ];
  load_rows<T, NJ>(kr, kb, a.row, key0, len, a.D, true, c, g);
  if (a.parents) build_tree(tree, a.parents + (int64_t)b * a.N, a.N);
  if (any) put(first, 0);
  __syncthreads();

  float acc = 0.f;
  for (int t = first, buf = 0; 16 * t < a.R; ++t, buf ^= 1) {
    const bool more = 16 * (t + 1) < a.R;
    if (more) fetch(t + 1);
    f32x4 qr[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) qr[j] = q_s[buf][64 * j + lane];
    const f32x4 s = score_tile<NJ, 2>(qr, kr);
    const f32x4 lse = *reinterpret_cast<const f32x4*>(&lse_s[buf][4 * g]);
    const int4 tok = *reinterpret_cast<const int4*>(&tok_s[buf][4 * g]);
    const int token[4] = {tok.x, tok.y, tok.z, tok.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = exp2f(fmaf(s[i], a.sl2, -lse[i]));
      bool sees = token[i] >= 0;
      if (a.parents) {
        const int at = max(token[i], 0), bit = nkey < 0 ? at : min(nkey, a.N - 1);
        sees = sees && (tree.seen[at][bit >> 5] >> (bit & 31) & 1);
      } else {
        sees = sees && nkey <= token[i];
      }
      acc += sees ? p : 0.f;
    }
    if (more) put(t + 1, buf ^ 1);
    __syncthreads();
  }
  acc = group4_sum(acc);
  if (g == 0 && key < len) {
    const int64_t at = ((int64_t)b * a.Hkv + hk) * a.C + key;
    a.w_out[at] = (a.w && key < past ? a.w[at] : 0.f) + acc;
  }
}

// Which of the new tokens (at most 64) each of them sees, one bit each, 0 for
// one that is not there.  By the first wave of a workgroup; no barrier.
__device__ __forceinline__ void build_bits(uint64_t* seen, int* par, const int32_t* parents, int N,
                                           int there) {
  const int i = threadIdx.x;
  if (i >= 64) return;
  uint64_t bits = 0;
  bool ok = i < min(N, there);
  if (parents == nullptr) {
    bits = ~0ull >> (63 - i);
  } else {
    par[i] = i < N ? parents[i] : -2;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    for (int at = i; ok;) {  // at falls with every step
      bits |= 1ull << at;
      const int p = par[at];
      if (p == -1) break;
      ok = p >= 0 && p < at;
      at = p;
    }
  }
  seen[i] = ok ? bits : 0;
}

// The sequence of a workgroup: past rows, rows in all, tokens whose row lies in
// the cache; len = 0: there is no sequence.
struct Seq {
  int past, len, there;
};
__device__ __forceinline__ Seq seq_of(const WeightArgs& a, int b) {
  const int p = a.past[b];
  Seq s;
  s.past = min(p, a.C);
  s.len = p < 0 ? 0 : (int)min((int64_t)s.past + a.N, (int64_t)a.C);
  s.there = s.len - s.past;
  return s;
}

// ------------------------------------------------- bf16, up to 16 query rows --

// Few query rows: bound by the stream of K.  A wave holds the rows (Q as the A
// operand of S = Q K^T) and streams 64-key tiles straight into registers as the
// B operand, one tile ahead.  A lane then has one key and four rows of each
// product: the sum over rows is four adds and two lane swaps.  One-wave
// workgroups, the key ranges of a KV head next to each other.  One token of 32/8
// heads of 128 over 262,144 keys (537 MB): 101 us, 5.3 TB/s.
template <int D>
__global__ __launch_bounds__(64) void cache_weights_stream_kernel(WeightArgs a) {
  constexpr int KS = D / 32, MB = 4;
  __shared__ int par[64];
  __shared__ uint64_t seen[64];
  const int lane = threadIdx.x;
  const int c = lane & 15, g = lane >> 4;
  const int kblk = blockIdx.x % a.kblocks, rest = blockIdx.x / a.kblocks;
  const int hk = rest % a.Hkv, b = rest / a.Hkv;
  const Seq sq = seq_of(a, b);
  const int per = ((sq.len + 63) / 64 + a.kblocks - 1) / a.kblocks;  // tiles of a workgroup
  const int key00 = 64 * per * kblk;
  if (key00 >= sq.len) return;
  const int ntiles = min(per, (sq.len - key00 + 63) / 64);

  const uint16_t* kb = static_cast<const uint16_t*>(a.k) + b * a.seq + hk * a.head + 8 * g;
  auto kload = [&](int j, bf16x8 (&kr)[MB][KS]) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const int row = min(key00 + 64 * j + 16 * mb + c, sq.len - 1);
#pragma unroll
      for (int kk = 0; kk < KS; ++kk)
        kr[mb][kk] = (*reinterpret_cast<const bf16x8*>(kb + row * a.row + 32 * kk));
    }
  };
  bf16x8 kra[MB][KS], krb[MB][KS];
  kload(0, kra);
  build_bits(seen, par, a.parents ? a.parents + (int64_t)b * a.N : nullptr, a.N, sq.there);
  __syncthreads();

  // Row c as A operand; the statistics of rows 4 g + i.
  bf16x8 qreg[KS];
  {
    const int rr = c < a.R ? c : 0;
    const int64_t qi = ((int64_t)b * a.N + rr / a.group) * a.Hq + hk * a.group + rr % a.group;
    const uint16_t* qrow = static_cast<const uint16_t*>(a.q) + qi * D;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) qreg[kk] = *reinterpret_cast<const bf16x8*>(qrow + 32 * kk + 8 * g);
  }
  float lse[4];
  uint64_t bits[4];  // tokens the row sees; 0: it gives nothing
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rs = 4 * g + i, rt = rs < a.R ? rs : 0;
    const int tk = rt / a.group;
    const int64_t si = ((int64_t)b * a.Hq + hk * a.group + rt % a.group) * a.N + tk;
    const float m = a.m[si], l = a.l[si];
    lse[i] = row_lse(m, l);
    bits[i] = rs < a.R && gives(m, l) ? seen[tk] : 0;
  }

  const int64_t wrow = ((int64_t)b * a.Hkv + hk) * a.C;
  auto tile = [&](int j, bf16x8 (&kc)[MB][KS], bf16x8 (&kn)[MB][KS]) {
    const int key0 = key00 + 64 * j;
    // (Loads complete in order: this one ahead of the next tile's.)
    const float before = a.w != nullptr && key0 + lane < sq.past ? a.w[wrow + key0 + lane] : 0.f;
    if (j + 1 < ntiles) kload(j + 1, kn);
    float sum[MB] = {0.f, 0.f, 0.f, 0.f};
    f32x4 s[MB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) s[mb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < KS; ++kk)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) s[mb] = mfma16x16x32(qreg[kk], kc[mb][kk], s[mb]);
    const bool own = key0 + 64 > sq.past;  // new tokens' rows among the keys
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        const float p = fast_exp2(fmaf(s[mb][i], a.sl2, -lse[i]));
        bool sees = bits[i] != 0;
        if (own) {
          const int nkey = key0 + 16 * mb + c - sq.past;
          if (nkey >= 0) sees = nkey < 64 && (bits[i] >> nkey & 1);
        }
        sum[mb] += sees ? p : 0.f;
      }
    // Lane 16 mb + c takes key 16 mb + c.
    float w = 0.f;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const float x = group4_sum(sum[mb]);
      if (g == mb) w = x;
    }
    if (key0 + lane < sq.len) a.w_out[wrow + key0 + lane] = before + w;
  };
  for (int j = 0; j < ntiles; j += 2) {
    tile(j, kra, krb);
    if (j + 1 < ntiles) tile(j + 1, krb, kra);
  }
}

// ---------------------------------------------- bf16, 17 to 256 query rows --

// A tile of 32 query rows in LDS, rows of 2 D bytes: head_dim 128 as
// tile128.h; head_dim 64: chunk L of row r at L ^ ((r >> 1) & 7), which gives
// the sixteen lanes of a read cycle (rows {0-3, 12-15, 20-27} or {4-11, 16-19,
// 28-31}) distinct chunks of the two rows that share 256 bytes of banks.
template <int D>
struct QTile {
  static constexpr int kBytes = 32 * 2 * D;
  static constexpr int kLanes = D / 8;       // lanes (16-byte chunks) of a row
  static constexpr int kRows = 64 / kLanes;  // rows of a wave instruction
  static __device__ __forceinline__ int swz(int r) { return D == 128 ? t128::swz(r) : r >> 1 & 7; }
  static __device__ __forceinline__ int off(int r, int chunk) { return r * 2 * D + 16 * (chunk ^ swz(r)); }
};

// All query rows of the KV head (at most 64 tokens) stay in LDS and the keys
// stream past them, 64 to a wave, in registers one tile ahead; no barrier after
// the start.  S = Q K^T (32 x 32 x 16): a lane has one key and 16 rows of each
// product, whose statistics are broadcast from LDS.  Rows that give nothing are
// zeros; a tile of such rows alone is left out, and one that has some of them
// selects (an infinite key makes their scores NaN).  32/8 heads of 128 over
// 262,000 keys: 8 tokens 118 us (4.5 TB/s), 26 130, 64 164 (670 TFLOP/s), of which
// five are padding 178, 171 without the selection.  Non-temporal loads of K, which
// each workgroup reads once too, took 182 there.
constexpr int kHeldRows = 256;
// With two 64-key tiles or fewer for each of the chip's 1,024 waves the rows
// pass by the keys faster than the keys by more than 64 rows (32/8 heads of 128:
// 64 tokens over 4,000 keys 13.1 us against 22.3, 26 over 16,000 17.4 against
// 18.9); with more keys not (26 over 32,000 28.7 against 23.8, 64 over 262,000 252
// against 164), nor with fewer rows (16 tokens over 4,000 keys 11.4 against 10.0).
constexpr int64_t kFewKeys = 1 << 17;
template <int D>
__global__ __launch_bounds__(256, 2) void cache_weights_rows_kernel(WeightArgs a) {
  using Q = QTile<D>;
  constexpr int KS = D / 16;
  __shared__ __attribute__((aligned(1024))) uint8_t qbuf[kHeldRows / 32 * Q::kBytes];
  __shared__ __attribute__((aligned(16))) float lse_s[kHeldRows];
  __shared__ __attribute__((aligned(16))) uint64_t bits_s[kHeldRows];
  __shared__ uint64_t seen[64];
  __shared__ int par[64];
  __shared__ int live_s, dead_s;  // a bit for each tile of 32 rows that has some that give something, nothing
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kc = lane & 31, hh = lane >> 5;
  const int kblk = blockIdx.x % a.kblocks, rest = blockIdx.x / a.kblocks;
  const int hk = rest % a.Hkv, b = rest / a.Hkv;
  const Seq sq = seq_of(a, b);
  const int all = (sq.len + 63) / 64;
  const int per = (all + a.kblocks - 1) / a.kblocks;  // tiles of a workgroup
  const int j0 = per * kblk + wave, j1 = min(per * (kblk + 1), all);
  if (per * kblk >= all) return;  // the whole workgroup

  const uint16_t* kb = static_cast<const uint16_t*>(a.k) + b * a.seq + hk * a.head + 8 * hh;
  auto kload = [&](int j, bf16x8 (&kr)[2][KS]) {
#pragma unroll
    for (int mb = 0; mb < 2; ++mb) {
      const int row = min(64 * j + 32 * mb + kc, sq.len - 1);
#pragma unroll
      for (int t = 0; t < KS; ++t)
        kr[mb][t] = (*reinterpret_cast<const bf16x8*>(kb + row * a.row + 16 * t));
    }
  };
  bf16x8 kra[2][KS], krb[2][KS];
  if (j0 < j1) kload(j0, kra);

  build_bits(seen, par, a.parents ? a.parents + (int64_t)b * a.N : nullptr, a.N, sq.there);
  if (threadIdx.x == 0) live_s = dead_s = 0;
  __syncthreads();
  const int tiles = (a.R + 31) / 32;
  {  // a row of each thread
    const int r = threadIdx.x, rr = r < a.R ? r : 0;
    const int tk = rr / a.group;
    const int64_t si = ((int64_t)b * a.Hq + hk * a.group + rr % a.group) * a.N + tk;
    const float m = a.m[si], l = a.l[si];
    const uint64_t bits = r < a.R && gives(m, l) ? seen[tk] : 0;
    lse_s[r] = bits != 0 ? row_lse(m, l) : INFINITY;
    bits_s[r] = bits;
    atomicOr(bits != 0 ? &live_s : &dead_s, 1 << (r >> 5));
  }
  __syncthreads();
  for (int x = threadIdx.x; x < 32 * tiles * Q::kLanes; x += 256) {
    const int r = x / Q::kLanes, ch = x % Q::kLanes;
    uint4 v = {0u, 0u, 0u, 0u};
    if (bits_s[r] != 0) {
      const int64_t qi = ((int64_t)b * a.N + r / a.group) * a.Hq + hk * a.group + r % a.group;
      v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + qi * D + 8 * ch);
    }
    *reinterpret_cast<uint4*>(qbuf + (r >> 5) * Q::kBytes + Q::off(r & 31, ch)) = v;
  }
  __syncthreads();
  const int live = __builtin_amdgcn_readfirstlane(live_s);
  const int whole = ~__builtin_amdgcn_readfirstlane(dead_s);

  int qoff[KS];
#pragma unroll
  for (int x = 0; x < KS; ++x) qoff[x] = Q::off(kc, 2 * x + hh);
  const int64_t wrow = ((int64_t)b * a.Hkv + hk) * a.C;
  auto keys = [&](int j, bf16x8 (&kr)[2][KS], bf16x8 (&kn)[2][KS]) {
    const int key0 = 64 * j;
    const float before = a.w != nullptr && key0 + lane < sq.past ? a.w[wrow + key0 + lane] : 0.f;
    if (j + 4 < j1) kload(j + 4, kn);
    float sum[2][4] = {};
    for (int t = 0; t < tiles; ++t) {
      if (!(live >> t & 1)) continue;
      const uint8_t* qt = qbuf + t * Q::kBytes;
      f32x16 s[2];
      s[0] = s[1] = f32x16{};
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        const bf16x8 qx = *reinterpret_cast<const bf16x8*>(qt + qoff[x]);
        s[0] = mfma32x32x16(qx, kr[0][x], s[0]);
        s[1] = mfma32x32x16(qx, kr[1][x], s[1]);
      }
      f32x4 lse[4];  // rows 8 w + 4 hh .. + 3
#pragma unroll
      for (int w = 0; w < 4; ++w) lse[w] = *reinterpret_cast<const f32x4*>(lse_s + 32 * t + 8 * w + 4 * hh);
      if (key0 + 64 <= sq.past) {
        auto add = [&](auto select) {
#pragma unroll
          for (int v = 0; v < 16; ++v)
#pragma unroll
            for (int mb = 0; mb < 2; ++mb) {
              const float x = lse[v >> 2][v & 3];
              const float p = fast_exp2(fmaf(s[mb][v], a.sl2, -x));
              sum[mb][v & 3] += decltype(select)::value && x == INFINITY ? 0.f : p;
            }
        };
        if (whole >> t & 1) add(std::false_type{});
        else add(std::true_type{});
      } else {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const uint64_t bits = bits_s[32 * t + 8 * (v >> 2) + 4 * hh + (v & 3)];
#pragma unroll
          for (int mb = 0; mb < 2; ++mb) {
            const float p = fast_exp2(fmaf(s[mb][v], a.sl2, -lse[v >> 2][v & 3]));
            const int nkey = key0 + 32 * mb + kc - sq.past;
            const bool sees = nkey < 0 ? bits != 0 : nkey < 64 && (bits >> nkey & 1);
            sum[mb][v & 3] += sees ? p : 0.f;
          }
        }
      }
    }
    // Lane 32 mb + kc takes key 32 mb + kc.
    float w[2];
#pragma unroll
    for (int mb = 0; mb < 2; ++mb) w[mb] = xor32_sum((sum[mb][0] + sum[mb][1]) + (sum[mb][2] + sum[mb][3]));
    if (key0 + lane < sq.len) a.w_out[wrow + key0 + lane] = before + (hh ? w[1] : w[0]);
  };
  for (int j = j0; j < j1; j += 8) {
    keys(j, kra, krb);
    if (j + 4 < j1) keys(j + 4, krb, kra);
  }
}

// ------------------------------------------------------- bf16, many tokens --

// Many query rows: bound by the exponentials and the products beside them.
// Workgroup: 256 keys of one KV head, 64 of each wave in registers (the A
// operand of S^T = K Q^T); the tokens of one query head after the other pass
// through LDS, kTok at a time, two buffers.  A lane has one query row and 16
// keys of each product, so a row's statistics are one register and a key's sum
// stays in its lane until the end.  512 tokens of 32/8 heads of 128 behind 32,000
// keys: 154 us, 880 TFLOP/s.
template <int D>
__global__ __launch_bounds__(256, 2) void cache_weights_tile_kernel(WeightArgs a) {
  using Q = QTile<D>;
  constexpr int KS = D / 16;
  constexpr int kTok = 128;                        // tokens of a chunk
  constexpr int kTiles = kTok / 32;
  constexpr int kInst = 32 / Q::kRows / 4;         // Q loads of a wave per 32 tokens
  constexpr int kPitch = 33;
  constexpr int kQBytes = 2 * kTiles * Q::kBytes, kPartBytes = 4 * 64 * kPitch * 4;
  // The Q buffers, then (after the walk) the lanes' sums.
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kQBytes > kPartBytes ? kQBytes : kPartBytes];
  __shared__ float lse_s[2][kTok];
  __shared__ Tree tree;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kc = lane & 31, hh = lane >> 5;
  const int kblk = a.kblocks - 1 - blockIdx.x % a.kblocks, rest = blockIdx.x / a.kblocks;
  const int hk = rest % a.Hkv, b = rest / a.Hkv;
  const Seq sq = seq_of(a, b);
  if (256 * kblk >= sq.len) return;  // the whole workgroup

  // Keys 32 mb + kc of the wave, dims 16 t + 8 hh.
  const int key0 = 256 * kblk + 64 * wave;
  const uint16_t* kb = static_cast<const uint16_t*>(a.k) + b * a.seq + hk * a.head + 8 * hh;
  bf16x8 kreg[2][KS];
#pragma unroll
  for (int mb = 0; mb < 2; ++mb) {
    const int row = min(key0 + 32 * mb + kc, sq.len - 1);
#pragma unroll
    for (int t = 0; t < KS; ++t)
      kreg[mb][t] = (*reinterpret_cast<const bf16x8*>(kb + row * a.row + 16 * t));
  }
  if (a.parents != nullptr) build_tree(tree, a.parents + (int64_t)b * a.N, a.N);

  // Chunks: kTok tokens of a head from `from` on (a chain's tokens before the
  // first that sees one of the workgroup's keys see none), then the next head.
  const int from = a.parents ? 0 : max(0, 256 * kblk - sq.past) / 32 * 32;
  const int per_head = sq.there > from ? (sq.there - from + kTok - 1) / kTok : 0;
  const int nchunks = per_head * a.group;
  const uint16_t* qb = static_cast<const uint16_t*>(a.q) + ((int64_t)b * a.N * a.Hq + (int64_t)hk * a.group) * D;
  const int64_t qtok = (int64_t)a.Hq * D;
  const int64_t sb = ((int64_t)b * a.Hq + hk * a.group) * a.N;
  uint32_t off[kInst];  // byte offset of the lane's 16 bytes from the first token's row
#pragma unroll
  for (int i = 0; i < kInst; ++i) {
    const int r = (wave * kInst + i) * Q::kRows + lane / Q::kLanes;
    off[i] = (uint32_t)(r * qtok * 2 + 16 * ((lane % Q::kLanes) ^ Q::swz(r)));
  }
  struct At {
    int head, token;
  };
  auto next = [&](At x) {
    x.token += kTok;
    if (x.token >= sq.there) x = At{x.head + 1, from};
    return x;
  };
  auto qissue = [&](const At& x, int buf) {
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const int t0 = x.token + 32 * t;
      if (t0 >= sq.there) continue;
      const uint16_t* base = qb + (int64_t)x.head * D + t0 * qtok;
      const uint32_t dst = t128::lds_addr(smem) + (buf * kTiles + t) * Q::kBytes + wave * kInst * 1024;
      if (t0 + 32 <= a.N) {
#pragma unroll
        for (int i = 0; i < kInst; ++i) t128::dma_b128(base, off[i], dst + 1024 * i);
      } else {  // rows past the tokens re-read the last one's
#pragma unroll
        for (int i = 0; i < kInst; ++i) {
          const int r = (wave * kInst + i) * Q::kRows + lane / Q::kLanes;
          const int over = max(0, t0 + r - (a.N - 1));
          t128::dma_b128(reinterpret_cast<const uint8_t*>(base) + off[i] - over * qtok * 2, dst + 1024 * i);
        }
      }
    }
  };
  float m_next = 0.f, l_next = 0.f;  // statistics of token threadIdx.x of the next chunk
  auto stats = [&](const At& x) {
    if (threadIdx.x >= kTok) return;
    const int64_t si = sb + (int64_t)x.head * a.N + min(x.token + (int)threadIdx.x, a.N - 1);
    m_next = a.m[si];
    l_next = a.l[si];
  };
  auto put_stats = [&](const At& x, int buf) {  // inf: the row gives nothing
    if (threadIdx.x >= kTok) return;
    const int tk = x.token + threadIdx.x;
    bool ok = tk < sq.there && gives(m_next, l_next);
    if (a.parents != nullptr && ok) ok = tree.seen[tk][tk >> 5] >> (tk & 31) & 1;
    lse_s[buf][threadIdx.x] = ok ? row_lse(m_next, l_next) : INFINITY;
  };

  int qoff[KS];
#pragma unroll
  for (int x = 0; x < KS; ++x) qoff[x] = Q::off(kc, 2 * x + hh);
  f32x16 acc[2];
  acc[0] = acc[1] = f32x16{};
  auto chunk = [&](auto buf_tag, const At& x) {
    constexpr int kBuf = decltype(buf_tag)::value;
#pragma unroll 1
    for (int t = 0; t < kTiles; ++t) {
      const int t0 = x.token + 32 * t;
      if (t0 >= sq.there) break;
      if (a.parents == nullptr && key0 - sq.past > t0 + 31) continue;  // none sees the wave's keys
      const uint8_t* qt = smem + (kBuf * kTiles + t) * Q::kBytes;
      const float lse = lse_s[kBuf][32 * t + kc];
      f32x16 s[2];
      s[0] = s[1] = f32x16{};
#pragma unroll
      for (int y = 0; y < KS; ++y) {
        const bf16x8 qx = *reinterpret_cast<const bf16x8*>(qt + qoff[y]);
        s[0] = mfma32x32x16(kreg[0][y], qx, s[0]);
        s[1] = mfma32x32x16(kreg[1][y], qx, s[1]);
      }
      // Every row of the tile sees every key of the wave.
      const bool ok = lse != INFINITY;
      const bool plain = key0 + 64 <= sq.past || (a.parents == nullptr && key0 + 63 - sq.past <= t0);
      if (plain && __all(ok)) {
#pragma unroll
        for (int mb = 0; mb < 2; ++mb)
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[mb][v] += fast_exp2(fmaf(s[mb][v], a.sl2, -lse));
      } else {
        uint64_t bits = 0;  // bit y: the row sees key key0 + y
        if (ok) {
          const int tk = t0 + kc;
          const int at0 = key0 - sq.past;  // the first key as a token
          if (a.parents == nullptr) {
            const int last = tk - at0;  // the last key that the row sees
            bits = last < 0 ? 0 : ~0ull >> (63 - min(last, 63));
          } else {
            if (at0 < 0) bits = at0 <= -64 ? ~0ull : ~0ull >> (64 + at0);
#pragma unroll
            for (int y = 0; y < 3; ++y) {  // words of 32 tokens that meet the 64 keys
              const int w = (at0 >> 5) + y;
              if (w < 0 || w >= kWords) continue;
              const uint64_t word = tree.seen[tk][w];
              const int sh = 32 * w - at0;
              if (sh < 64) bits |= sh >= 0 ? word << sh : word >> -sh;
            }
          }
          bits >>= 4 * hh;
        }
#pragma unroll
        for (int mb = 0; mb < 2; ++mb)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const float p = fast_exp2(fmaf(s[mb][v], a.sl2, -lse));
            const bool sees = bits >> (32 * mb + 8 * (v >> 2) + (v & 3)) & 1;
            acc[mb][v] += sees ? p : 0.f;
          }
      }
    }
  };
  // Chunk c: its rows and statistics are in buffer c % 2; while it is computed,
  // the next chunk's rows go to the other buffer, its statistics to registers.
  At at{0, from};
  if (nchunks > 0) {
    qissue(at, 0);
    stats(at);
    put_stats(at, 0);
  }
  auto stage = [&](auto buf_tag, int c) {
    constexpr int kBuf = decltype(buf_tag)::value;
    t128::wait_vmem();
    __syncthreads();
    const At mine = at;
    at = next(at);
    if (c + 1 < nchunks) {
      qissue(at, kBuf ^ 1);
      stats(at);
    }
    chunk(buf_tag, mine);
    if (c + 1 < nchunks) put_stats(at, kBuf ^ 1);
  };
  for (int c = 0; c < nchunks; c += 2) {
    stage(std::integral_constant<int, 0>{}, c);
    if (c + 1 < nchunks) stage(std::integral_constant<int, 1>{}, c + 1);
  }
  // A key's sum over the 32 lanes of its half: through LDS, lane x takes key x.
  __syncthreads();  // the Q buffers are done with
  float* mp = reinterpret_cast<float*>(smem) + wave * 64 * kPitch;
#pragma unroll
  for (int mb = 0; mb < 2; ++mb)
#pragma unroll
    for (int v = 0; v < 16; ++v) mp[lane * kPitch + 16 * mb + v] = acc[mb][v];
  __syncthreads();
  const int key = key0 + lane;
  if (key >= sq.len) return;
  const int in = lane & 31;
  const float* src = mp + (in >> 2 & 1) * 32 * kPitch + 16 * (lane >> 5) + 4 * (in >> 3) + (in & 3);
  float w = 0.f;
#pragma unroll
  for (int x = 0; x < 32; ++x) w += src[x * kPitch];
  const int64_t wi = ((int64_t)b * a.Hkv + hk) * a.C + key;
  a.w_out[wi] = (a.w != nullptr && key < sq.past ? a.w[wi] : 0.f) + w;
}

}  // namespace

hipError_t launch_cache_weights(const CacheProblem& p, const void* q, const void* k,
                                const float* m, const float* l, const float* w, float* w_out,
                                hipStream_t st) {
  WeightArgs a;
  a.q = q;
  a.k = k;
  a.m = m;
  a.l = l;
  a.w = w;
  a.w_out = w_out;
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
  a.seq = p.seq;
  a.row = p.row;
  a.head = p.head;
  a.sl2 = p.sl2;
  auto launch = [&](auto kernel, int64_t kblocks, int threads) {
    a.kblocks = (int)kblocks;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(kblocks * p.Hkv * p.B)), dim3(threads), 0, st, a);
  };
  auto go = [&](auto kernel) { launch(kernel, (p.C + 63) / 64, 256); };
  auto by_dim = [&](auto t) {
    using T = decltype(t);
    if (p.D <= 16) go(cache_weights32_kernel<T, 1>);
    else if (p.D <= 32) go(cache_weights32_kernel<T, 2>);
    else if (p.D <= 64) go(cache_weights32_kernel<T, 4>);
    else if (p.D <= 96) go(cache_weights32_kernel<T, 6>);
    else if (p.D <= 128) go(cache_weights32_kernel<T, 8>);
    else go(cache_weights32_kernel<T, 16>);
  };
  auto bf16 = [&](auto d) {
    constexpr int kD = decltype(d)::value;
    const int64_t heads = (int64_t)p.B * p.Hkv, tiles = (p.C + 63) / 64;
    // As many workgroups as the chip holds, in which the lengths are dealt out.
    // Up to 16 rows: one token over 262,000 keys 107 us against 117 with the rows
    // in LDS, four over 4,000 5.6 against 6.5.
    if (a.R <= 16)
      launch(cache_weights_stream_kernel<kD>, std::min(std::max<int64_t>(1, 2048 / heads), tiles), 64);
    else if (a.R <= kHeldRows && p.N <= 64 && (a.R <= 64 || heads * p.C > kFewKeys))
      launch(cache_weights_rows_kernel<kD>, std::min(std::max<int64_t>(1, 512 / heads), (tiles + 3) / 4), 256);
    else
      launch(cache_weights_tile_kernel<kD>, (p.C + 255) / 256, 256);
  };
  // Without tokens q may be null; the tile kernel's row offsets are 32-bit.
  const bool mfma = p.dtype == 1 && !p.precise && p.N > 0 && (int64_t)p.Hq * p.D < 1 << 25;
  if (mfma && p.D == 128) bf16(std::integral_constant<int, 128>{});
  else if (mfma && p.D == 64) bf16(std::integral_constant<int, 64>{});
  else if (p.dtype == 1) by_dim(uint16_t{});
  else by_dim(float{});
  return hipGetLastError();
}

}  // namespace lc
