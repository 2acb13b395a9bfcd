// Accumulated attention weight of the rows of a KV cache (gfx950): with the
// statistics of the attention given,
//   w[h][j] = sum over the query rows r of KV head h that see row j of
//             exp(s_rj - m_r) / l_r = sum exp2(s'_rj - lse2_r),
// s' in log2 units and lse2 = m log2(e) + log2(l), so that a row costs one
// subtraction and one exp2 per key.  Keys are stationary and the query rows
// stream past them, which makes the sum over rows a sum within a lane: no
// atomics, a fixed order.  Rows that a key is not seen by are left out by
// selection, not by a factor, so a NaN in an unseen place stays there.
#include "common.h"
#include "cache.h"
#include "kernels.h"
#include "tile32.h"

namespace lc {
namespace {

struct WeightArgs {
  const void *q, *k;
  const float *m, *l, *w;
  float* w_out;
  const int32_t *past, *parents;
  int B, N, C, Hq, Hkv, D, group, R, kblocks;
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

// fp32 products, any head_dim: a wave holds 16 keys and walks the query rows
// of its KV head, (token, head of the group) by token, 16 at a time.
template <typename T, int NJ>
__global__ __launch_bounds__(256) void cache_weights32_kernel(WeightArgs a) {
  __shared__ Tree tree;
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
  if (a.parents) build_tree(tree, a.parents + (int64_t)b * a.N, a.N);

  const int key0 = 64 * kblk + 16 * wave;
  const int key = key0 + c;
  const int nkey = key - past;  // the token whose row this is, if >= 0
  const T* kb = static_cast<const T*>(a.k) + b * a.seq + hk * a.head;
  f32x4 kr[NJ];
  load_rows<T, NJ>(kr, kb, a.row, key0, len, a.D, true, c, g);

  const T* qb = static_cast<const T*>(a.q) + ((int64_t)b * a.N * a.Hq + (int64_t)hk * a.group) * a.D;
  const int64_t sb = ((int64_t)b * a.Hq + hk * a.group) * a.N;
  float acc = 0.f;
  // A chain's rows before the first token that sees one of the keys see none.
  const int first = a.parents ? 0 : max(0, key0 - past) * a.group / 16;
  for (int t = first; 16 * t < a.R; ++t) {
    f32x4 qr[NJ];
    {
      const int r = 16 * t + c, rr = r < a.R ? r : 0;
      const T* qp = qb + ((int64_t)(rr / a.group) * a.Hq + rr % a.group) * a.D;
#pragma unroll
      for (int j = 0; j < NJ; ++j) qr[j] = load_w<T, 4>(qp, r < a.R ? 16 * j + 4 * g : a.D, a.D, true);
    }
    const f32x4 s = score_tile<NJ, 2>(qr, kr);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * t + 4 * g + i, rr = r < a.R ? r : 0;
      const int token = rr / a.group;
      const int64_t si = sb + (int64_t)(rr - token * a.group) * a.N + token;
      const float m = a.m[si], l = a.l[si];
      const float p = exp2f(fmaf(s[i], a.sl2, -fmaf(m, kLog2e, log2f(l))));
      bool sees = r < a.R && token < there && l > 0.f && m != -INFINITY;
      if (a.parents) {
        const int bit = nkey < 0 ? token : min(nkey, a.N - 1);
        sees = sees && (tree.seen[token][bit >> 5] >> (bit & 31) & 1);
      } else {
        sees = sees && nkey <= token;
      }
      acc += sees ? p : 0.f;
    }
  }
  acc = group4_sum(acc);
  if (g == 0 && key < len) {
    const int64_t at = ((int64_t)b * a.Hkv + hk) * a.C + key;
    a.w_out[at] = (a.w && key < past ? a.w[at] : 0.f) + acc;
  }
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
  a.kblocks = (p.C + 63) / 64;
  a.seq = p.seq;
  a.row = p.row;
  a.head = p.head;
  a.sl2 = p.sl2;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(a.kblocks * p.Hkv * p.B)), dim3(256), 0, st, a);
  };
  auto by_dim = [&](auto t) {
    using T = decltype(t);
    if (p.D <= 16) go(cache_weights32_kernel<T, 1>);
    else if (p.D <= 32) go(cache_weights32_kernel<T, 2>);
    else if (p.D <= 64) go(cache_weights32_kernel<T, 4>);
    else if (p.D <= 96) go(cache_weights32_kernel<T, 6>);
    else if (p.D <= 128) go(cache_weights32_kernel<T, 8>);
    else go(cache_weights32_kernel<T, 16>);
  };
  if (p.dtype == 1) by_dim(uint16_t{});
  else by_dim(float{});
  return hipGetLastError();
}

}  // namespace lc
