// C-ABI entry points of the KV-cache operators (include/longctx100m_attn.h).
// The reference keeps no cache (src/longctx100m/distributed_infer.py:185-219
// recomputes the prefill for every token), so these have no counterpart there.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "longctx100m_attn.h"
#include "cache.h"
#include "kernels.h"

namespace {

using lc::hip_error;
using lc::set_error;

size_t elem_size(const lc_cache_t* c) { return c->dtype == LC_DTYPE_BF16 ? 2 : 4; }

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

struct Range {
  uintptr_t lo, hi;
};
Range range(const void* p, size_t bytes) {
  const auto b = reinterpret_cast<uintptr_t>(p);
  return Range{b, p ? b + bytes : b};
}
bool meet(Range a, Range b) { return a.lo < b.hi && b.lo < a.hi; }
// An output that is its input, or lies apart from it.
bool same_or_apart(const void* in, const void* out, size_t bytes) {
  return in == out || !meet(range(in, bytes), range(out, bytes));
}

// written: rows of the cache are written, so no two may share memory.
int check_cache(const lc_cache_t* c, bool written, bool queries) {
  if (!c) return set_error(LC_ERR_INVALID, "null cache argument");
  if (c->batch <= 0 || c->tokens < 0 || c->capacity <= 0 || c->heads_kv <= 0 || c->head_dim <= 0 ||
      (queries && c->heads_q <= 0))
    return set_error(LC_ERR_INVALID, "a cache needs batch, capacity, heads and head_dim > 0 and tokens >= 0");
  if (queries && c->heads_q % c->heads_kv != 0)
    return set_error(LC_ERR_INVALID, "heads_q (%d) must be a multiple of heads_kv (%d)", c->heads_q,
                     c->heads_kv);
  if (c->dtype != LC_DTYPE_F32 && c->dtype != LC_DTYPE_BF16)
    return set_error(LC_ERR_UNSUPPORTED, "unsupported dtype %d", c->dtype);
  if (c->flags & ~LC_FLAG_PRECISE)
    return set_error(LC_ERR_INVALID, "unknown flag bits 0x%x", c->flags & ~LC_FLAG_PRECISE);
  if (c->head_dim % 16 != 0 || c->head_dim > 256)
    return set_error(LC_ERR_UNSUPPORTED, "the cache operators need head_dim %% 16 == 0 and <= 256");
  // A launch holds fewer than 2^32 threads in a dimension, and row indices of
  // one sequence's queries are 32-bit.
  const int64_t heads = (int64_t)c->batch * c->heads_kv;
  if (heads > 1 << 21 || heads * ((c->capacity + 63LL) / 64) > 1 << 23 ||
      (queries && (int64_t)c->batch * c->heads_q > 1 << 24) ||
      (queries && (int64_t)c->tokens * c->heads_q > 1 << 30))
    return set_error(LC_ERR_UNSUPPORTED, "the cache or its queries exceed the kernels' grids");
  const int64_t e = 16 / (int64_t)elem_size(c);
  if (c->seq_stride < 0 || c->row_stride < 0 || c->head_stride < 0 || c->seq_stride % e ||
      c->row_stride % e || c->head_stride % e)
    return set_error(LC_ERR_INVALID, "cache strides must be multiples of 16 bytes");
  if (c->row_stride > (int64_t)1 << 24)
    return set_error(LC_ERR_UNSUPPORTED, "cache rows lie more than 2^24 elements apart");
  if (c->seq_stride > (int64_t)1 << 40 || c->head_stride > (int64_t)1 << 40)
    return set_error(LC_ERR_UNSUPPORTED, "sequences or heads lie more than 2^40 elements apart");
  if (written) {
    struct Dim {
      int64_t stride, n;
    } d[3] = {{c->seq_stride, c->batch}, {c->row_stride, c->capacity}, {c->head_stride, c->heads_kv}};
    std::sort(d, d + 3, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
    int64_t extent = c->head_dim;
    for (const Dim& x : d) {
      if (x.n == 1) continue;
      if (x.stride < extent)
        return set_error(LC_ERR_INVALID, "rows of a cache that is written must not overlap");
      extent += x.stride * (x.n - 1);
    }
  }
  return LC_OK;
}

lc::CacheProblem make_problem(const lc_cache_t* c, const int32_t* past, const int32_t* parents) {
  lc::CacheProblem p;
  p.B = c->batch;
  p.N = c->tokens;
  p.C = c->capacity;
  p.Hq = c->heads_q;
  p.Hkv = c->heads_kv;
  p.D = c->head_dim;
  p.dtype = c->dtype;
  p.precise = (c->flags & LC_FLAG_PRECISE) != 0;
  p.seq = c->seq_stride;
  p.row = c->row_stride;
  p.head = c->head_stride;
  p.past = past;
  p.parents = parents;
  p.sl2 = (float)(std::pow((double)p.D, -0.5) * 1.4426950408889634);
  return p;
}

int check_attn(const lc_cache_t* c) {
  if (int rc = check_cache(c, false, true)) return rc;
  if (c->tokens > LC_CACHE_MAX_TOKENS)
    return set_error(LC_ERR_UNSUPPORTED, "at most %d new tokens", LC_CACHE_MAX_TOKENS);
  if ((int64_t)c->batch * c->heads_q * c->tokens > 1 << 22)
    return set_error(LC_ERR_UNSUPPORTED, "the cache or its queries exceed the kernels' grids");
  return LC_OK;
}

}  // namespace

extern "C" {

size_t lc_cache_attn_workspace_bytes(const lc_cache_t* cache) {
  if (check_attn(cache) || cache->tokens == 0) return 0;
  return lc::cache_attn_bytes(make_problem(cache, nullptr, nullptr));
}

int lc_cache_attn(const lc_cache_t* cache, const int32_t* past, const int32_t* parents,
                  const void* q, const void* k, const void* v, void* out, float* m, float* l,
                  void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_attn(cache)) return rc;
  if (cache->tokens == 0) return LC_OK;
  if (!past || !q || !k || !v || !out) return set_error(LC_ERR_INVALID, "null pointer argument");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16))
    return set_error(LC_ERR_INVALID, "q, k, v and out must be 16-byte aligned");
  if (!aligned(past, 4) || !aligned(parents, 4) || !aligned(m, 4) || !aligned(l, 4))
    return set_error(LC_ERR_INVALID, "past, parents, m and l must be 4-byte aligned");
  const lc::CacheProblem p = make_problem(cache, past, parents);
  const size_t need = lc::cache_attn_bytes(p);
  if (workspace_bytes < need || !workspace)
    return set_error(LC_ERR_WORKSPACE, "cache attention needs a workspace of %zu bytes, got %zu", need,
                     workspace ? workspace_bytes : (size_t)0);
  if (!aligned(workspace, 16))
    return set_error(LC_ERR_INVALID, "the workspace must be 16-byte aligned");
  hipError_t e = lc::launch_cache_attn(p, q, k, v, out, m, l, workspace,
                                       static_cast<hipStream_t>(stream));
  return e == hipSuccess ? LC_OK : hip_error(e, "lc_cache_attn launch");
}

int lc_cache_weights(const lc_cache_t* cache, const int32_t* past, const int32_t* parents,
                     const void* q, const void* k, const float* m, const float* l,
                     const float* weights, float* weights_out, void* stream) {
  if (int rc = check_cache(cache, false, true)) return rc;
  if (parents && cache->tokens > LC_CACHE_MAX_TOKENS)
    return set_error(LC_ERR_UNSUPPORTED, "at most %d new tokens with parents", LC_CACHE_MAX_TOKENS);
  if (!past || !k || !weights_out || (cache->tokens > 0 && (!q || !m || !l)))
    return set_error(LC_ERR_INVALID, "null pointer argument");
  if (!aligned(q, 16) || !aligned(k, 16))
    return set_error(LC_ERR_INVALID, "q and k must be 16-byte aligned");
  if (!aligned(past, 4) || !aligned(parents, 4) || !aligned(m, 4) || !aligned(l, 4) ||
      !aligned(weights, 4) || !aligned(weights_out, 4))
    return set_error(LC_ERR_INVALID, "past, parents, m, l and the weights must be 4-byte aligned");
  const size_t wb = (size_t)cache->batch * cache->heads_kv * cache->capacity * sizeof(float);
  if (!same_or_apart(weights, weights_out, wb))
    return set_error(LC_ERR_INVALID, "weights_out must be weights or not overlap it");
  hipError_t e = lc::launch_cache_weights(make_problem(cache, past, parents), q, k, m, l, weights,
                                          weights_out, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? LC_OK : hip_error(e, "lc_cache_weights launch");
}

size_t lc_cache_evict_workspace_bytes(const lc_cache_t* cache) {
  if (check_cache(cache, true, false)) return 0;
  return lc::cache_evict_bytes(cache->batch, cache->heads_kv, cache->capacity);
}

int lc_cache_evict(const lc_cache_t* cache, int32_t budget, int32_t sinks, int32_t recent,
                   const int32_t* lens, const int32_t* kept, const int32_t* ends, void* k, void* v,
                   const float* weights, const int32_t* positions, float* weights_out,
                   int32_t* positions_out, int32_t* lens_out, void* workspace,
                   size_t workspace_bytes, void* stream) {
  if (int rc = check_cache(cache, true, false)) return rc;
  if (budget <= 0) return set_error(LC_ERR_INVALID, "budget must be positive");
  if (sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
    return set_error(LC_ERR_INVALID, "sinks and recent must be >= 0 and fit the budget together");
  if (!lens || !k || !v || !weights || !weights_out || !positions_out || !lens_out)
    return set_error(LC_ERR_INVALID, "null pointer argument");
  if (kept && !positions)
    return set_error(LC_ERR_INVALID, "kept rows need their positions");
  if (!aligned(k, 16) || !aligned(v, 16))
    return set_error(LC_ERR_INVALID, "k and v must be 16-byte aligned");
  for (const void* p : {(const void*)lens, (const void*)kept, (const void*)ends, (const void*)weights,
                        (const void*)positions, (const void*)weights_out,
                        (const void*)positions_out, (const void*)lens_out})
    if (!aligned(p, 4))
      return set_error(LC_ERR_INVALID, "lengths, weights and positions must be 4-byte aligned");
  const size_t n = (size_t)cache->batch * cache->heads_kv * cache->capacity * 4;
  if (!same_or_apart(weights, weights_out, n) || !same_or_apart(positions, positions_out, n))
    return set_error(LC_ERR_INVALID, "weights_out and positions_out must be their inputs or not overlap them");
  const size_t nb = (size_t)cache->batch * 4;
  const Range lo = range(lens_out, nb), wo = range(weights_out, n), po = range(positions_out, n);
  const Range lens_in[3] = {range(lens, nb), range(kept, nb), range(ends, nb)};
  for (const Range& r : lens_in)
    if (meet(lo, r) || meet(wo, r) || meet(po, r))
      return set_error(LC_ERR_INVALID, "outputs must not overlap lens, kept or ends");
  if (meet(lo, wo) || meet(lo, po) || meet(wo, po) || meet(wo, range(positions, n)) ||
      meet(po, range(weights, n)) || meet(lo, range(weights, n)) || meet(lo, range(positions, n)))
    return set_error(LC_ERR_INVALID, "weights, positions and lengths must not overlap each other");
  const size_t need = lc::cache_evict_bytes(cache->batch, cache->heads_kv, cache->capacity);
  if (workspace_bytes < need || !workspace)
    return set_error(LC_ERR_WORKSPACE, "eviction needs a workspace of %zu bytes, got %zu", need,
                     workspace ? workspace_bytes : (size_t)0);
  if (!aligned(workspace, 16))
    return set_error(LC_ERR_INVALID, "the workspace must be 16-byte aligned");
  lc::EvictProblem p;
  p.B = cache->batch;
  p.C = cache->capacity;
  p.Hkv = cache->heads_kv;
  p.D = cache->head_dim;
  p.elem = (int)elem_size(cache);
  p.seq = cache->seq_stride;
  p.row = cache->row_stride;
  p.head = cache->head_stride;
  p.budget = std::min(budget, cache->capacity);
  p.sinks = sinks;
  p.recent = recent;
  p.lens = lens;
  p.kept = kept;
  p.ends = ends;
  p.k = k;
  p.v = v;
  p.w = weights;
  p.pos = positions;
  p.w_out = weights_out;
  p.pos_out = positions_out;
  p.lens_out = lens_out;
  hipError_t e = lc::launch_cache_evict(p, workspace, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? LC_OK : hip_error(e, "lc_cache_evict launch");
}

int lc_cache_commit(const lc_cache_t* cache, int32_t layers, void* const* ks, void* const* vs,
                    const int32_t* past, const int32_t* path, int32_t* lens_out, void* stream) {
  if (int rc = check_cache(cache, true, false)) return rc;
  if (layers < 0) return set_error(LC_ERR_INVALID, "layers must be >= 0");
  if (!past || !lens_out || (cache->tokens > 0 && !path) || (layers > 0 && (!ks || !vs)))
    return set_error(LC_ERR_INVALID, "null pointer argument");
  for (int i = 0; i < layers; ++i) {
    if (!ks[i] || !vs[i]) return set_error(LC_ERR_INVALID, "null k or v of layer %d", i);
    if (!aligned(ks[i], 16) || !aligned(vs[i], 16))
      return set_error(LC_ERR_INVALID, "k and v must be 16-byte aligned");
    if (ks[i] == vs[i])  // its rows would be moved twice
      return set_error(LC_ERR_INVALID, "k and v of layer %d are the same cache", i);
  }
  if (!aligned(past, 4) || !aligned(path, 4) || !aligned(lens_out, 4))
    return set_error(LC_ERR_INVALID, "past, path and lens_out must be 4-byte aligned");
  const size_t nb = (size_t)cache->batch * 4;
  if (meet(range(lens_out, nb), range(past, nb)) ||
      meet(range(lens_out, nb), range(path, nb * cache->tokens)))
    return set_error(LC_ERR_INVALID, "lens_out must not overlap past or path");
  const size_t e = elem_size(cache);
  lc::CommitArgs a{};
  a.B = cache->batch;
  a.P = cache->tokens;
  a.C = cache->capacity;
  a.Hkv = cache->heads_kv;
  a.chunks = (int)(cache->head_dim * e / 16);
  a.seq = cache->seq_stride * (int64_t)e;
  a.row = cache->row_stride * (int64_t)e;
  a.head = cache->head_stride * (int64_t)e;
  a.past = past;
  a.path = path;
  int at = 0;
  do {  // the lengths also without layers
    const int n = std::min(layers - at, lc::kCommitLayers);
    for (int i = 0; i < n; ++i) {
      a.k[i] = static_cast<uint8_t*>(ks[at + i]);
      a.v[i] = static_cast<uint8_t*>(vs[at + i]);
    }
    a.lens_out = at == 0 ? lens_out : nullptr;
    hipError_t err = lc::launch_cache_commit(a, n, static_cast<hipStream_t>(stream));
    if (err != hipSuccess) return hip_error(err, "lc_cache_commit launch");
    at += n;
  } while (at < layers);
  return LC_OK;
}

}  // extern "C"
