// C-ABI entry points of rotary positions (include/longctx100m_layer.h) and of the
// paged 8-bit cache (include/longctx100m_attn.h).  The reference rotates by a
// table of consecutive positions (rust/longctx100m-model/src/rope.rs:101-127) and
// keeps no cache (src/longctx100m/distributed_infer.py:185-219).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "longctx100m_attn.h"
#include "longctx100m_layer.h"
#include "kernels.h"
#include "paged.h"
#include "rotary.h"

namespace {

using lc::hip_error;
using lc::set_error;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

struct Range {
  uintptr_t lo, hi;
};
Range range(const void* p, size_t bytes) {
  const auto b = reinterpret_cast<uintptr_t>(p);
  return Range{b, p ? b + bytes : b};
}
bool meet(Range a, Range b) { return a.lo < b.hi && b.lo < a.hi; }

// Rows of heads of a tensor [batch, tokens, heads, head_dim].
struct Rows {
  int64_t batch, tokens, heads, D;
  const lc_rows_t* s;
  size_t elem;

  // Elements from the first to behind the last: 2^40 at most (check).
  int64_t extent() const {
    return (batch - 1) * s->seq_stride + (tokens - 1) * s->token_stride + (heads - 1) * s->head_stride + D;
  }
  Range bytes(const void* p) const { return range(p, (size_t)extent() * elem); }
  // Whether every row is so aligned.
  bool vec(const void* p, int bytes = 16) const {
    const int64_t e = bytes / (int64_t)elem;
    return aligned(p, bytes) && (batch == 1 || s->seq_stride % e == 0) &&
           (tokens == 1 || s->token_stride % e == 0) && (heads == 1 || s->head_stride % e == 0);
  }
  int check(const char* name) const {
    if (!s) return set_error(LC_ERR_INVALID, "null strides of %s", name);
    const int64_t st[3] = {s->seq_stride, s->token_stride, s->head_stride};
    for (int64_t x : st)
      if (x < 0 || x > (int64_t)1 << 40)
        return set_error(LC_ERR_INVALID, "strides of %s must lie in 0 .. 2^40", name);
    const __int128 last = (__int128)(batch - 1) * st[0] + (__int128)(tokens - 1) * st[1] +
                          (__int128)(heads - 1) * st[2] + D;
    if (last > (__int128)1 << 40) return set_error(LC_ERR_INVALID, "%s spans more than 2^40 elements", name);
    return LC_OK;
  }
  // No two rows may share memory.
  int check_written(const char* name) const {
    struct Dim {
      int64_t stride, n;
    } d[3] = {{s->seq_stride, batch}, {s->token_stride, tokens}, {s->head_stride, heads}};
    std::sort(d, d + 3, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
    int64_t extent = D;
    for (const Dim& x : d) {
      if (x.n == 1) continue;
      if (x.stride < extent) return set_error(LC_ERR_INVALID, "rows of %s must not overlap", name);
      extent += x.stride * (x.n - 1);
    }
    return LC_OK;
  }
  bool same(const Rows& o) const {
    return (batch == 1 || s->seq_stride == o.s->seq_stride) &&
           (tokens == 1 || s->token_stride == o.s->token_stride) &&
           (heads == 1 || s->head_stride == o.s->head_stride);
  }
};

int check_dtype(int32_t dtype) {
  if (dtype != LC_DTYPE_F32 && dtype != LC_DTYPE_BF16)
    return set_error(LC_ERR_UNSUPPORTED, "unsupported dtype %d", dtype);
  return LC_OK;
}

int check_rotary(const lc_rotary_t* r) {
  if (!r) return set_error(LC_ERR_INVALID, "null rotary argument");
  if (r->head_dim <= 0 || r->head_dim > 256)
    return set_error(LC_ERR_UNSUPPORTED, "rotary positions need head_dim in 1 .. 256");
  if (r->rotary_dim <= 0 || r->rotary_dim % 2 != 0 || r->rotary_dim > r->head_dim)
    return set_error(LC_ERR_INVALID, "rotary_dim must be even, positive and at most head_dim");
  if (r->interleaved != 0 && r->interleaved != 1)
    return set_error(LC_ERR_INVALID, "interleaved must be 0 or 1");
  if (!std::isfinite(r->factor)) return set_error(LC_ERR_INVALID, "the rotary factor must be finite");
  if (!r->turns) return set_error(LC_ERR_INVALID, "null pointer argument");
  if (!aligned(r->turns, 8)) return set_error(LC_ERR_INVALID, "turns must be 8-byte aligned");
  return LC_OK;
}

lc::Turns make_turns(const lc_rotary_t* r) {
  lc::Turns t;
  t.turns = r ? r->turns : nullptr;
  t.half = r ? r->rotary_dim / 2 : 0;
  t.interleaved = r ? r->interleaved : 0;
  t.factor = r ? r->factor : 1.f;
  return t;
}

lc::HeadRows head_rows(const lc_rows_t* s) {
  return lc::HeadRows{s->seq_stride, s->token_stride, s->head_stride};
}

// A launch holds fewer than 2^32 threads in a dimension.
constexpr int64_t kMostGroups = (1 << 24) - 1;

int check_paged(const lc_paged_t* c, bool queries) {
  if (!c) return set_error(LC_ERR_INVALID, "null cache argument");
  if (c->batch <= 0 || c->tokens < 0 || c->heads_kv <= 0 || c->head_dim <= 0 || c->pages <= 0 ||
      c->table_width <= 0 || (queries && c->heads_q <= 0))
    return set_error(LC_ERR_INVALID,
                     "a paged cache needs batch, heads, head_dim, pages and table_width > 0 and tokens >= 0");
  if (queries && c->heads_q % c->heads_kv != 0)
    return set_error(LC_ERR_INVALID, "heads_q (%d) must be a multiple of heads_kv (%d)", c->heads_q,
                     c->heads_kv);
  if (queries && c->heads_q / c->heads_kv > 1 << 16)
    return set_error(LC_ERR_UNSUPPORTED, "more than 2^16 query heads share a KV head");
  if (int rc = check_dtype(c->dtype)) return rc;
  if (c->flags) return set_error(LC_ERR_INVALID, "unknown flag bits 0x%x", c->flags);
  if (c->head_dim % 16 != 0 || c->head_dim > 256)
    return set_error(LC_ERR_UNSUPPORTED, "the paged cache needs head_dim %% 16 == 0 and <= 256");
  if (c->page_rows != 16 && c->page_rows != 32 && c->page_rows != 64 && c->page_rows != 128)
    return set_error(LC_ERR_UNSUPPORTED, "a page has 16, 32, 64 or 128 rows");
  // (All sequences' 64-key tiles are counted in 31 bits, shared pages in each.)
  if ((int64_t)c->table_width * c->page_rows > 1 << 30 || (int64_t)c->batch * c->heads_kv > 1 << 20 ||
      (int64_t)c->table_width * c->page_rows * c->batch > (int64_t)1 << 36 ||
      c->tokens > 1 << 24 || (int64_t)c->batch * c->tokens * (queries ? c->heads_q : c->heads_kv) > 1 << 25)
    return set_error(LC_ERR_UNSUPPORTED, "the cache or its tokens exceed the kernels' grids");
  return LC_OK;
}

// Pages, scales, table, lengths; and what they occupy, to keep outputs apart.
struct PoolRanges {
  Range r[7];
};
int check_pool(const lc_paged_t* c, const int32_t* table, const int32_t* past, const int32_t* counts,
               const void* k, const void* v, const float* ks, const float* vs, PoolRanges* out) {
  if (!table || !past || !k || !v || !ks || !vs) return set_error(LC_ERR_INVALID, "null pointer argument");
  if (!aligned(k, 16) || !aligned(v, 16)) return set_error(LC_ERR_INVALID, "pages must be 16-byte aligned");
  if (!aligned(table, 4) || !aligned(past, 4) || !aligned(counts, 4) || !aligned(ks, 4) || !aligned(vs, 4))
    return set_error(LC_ERR_INVALID, "the table, lengths and scales must be 4-byte aligned");
  const size_t heads = (size_t)c->pages * c->heads_kv, bytes = heads * c->page_rows * c->head_dim;
  const size_t n = (size_t)c->batch * 4;
  *out = PoolRanges{{range(k, bytes), range(v, bytes), range(ks, heads * 4), range(vs, heads * 4),
                     range(table, n * c->table_width), range(past, n), range(counts, n)}};
  for (int i = 0; i < 4; ++i)
    for (int j = i + 1; j < 4; ++j)
      if (meet(out->r[i], out->r[j]))
        return set_error(LC_ERR_INVALID, "pages and scales of K and V must not overlap");
  return LC_OK;
}

lc::PagedProblem make_problem(const lc_paged_t* c, const int32_t* table, const int32_t* past,
                              const int32_t* counts, const void* k, const void* v, const float* ks,
                              const float* vs) {
  lc::PagedProblem p;
  p.B = c->batch;
  p.N = c->tokens;
  p.Hq = c->heads_q;
  p.dtype = c->dtype;
  p.pool.pages = c->pages;
  p.pool.rows = c->page_rows;
  p.pool.Hkv = c->heads_kv;
  p.pool.D = c->head_dim;
  p.pool.k = static_cast<uint8_t*>(const_cast<void*>(k));
  p.pool.v = static_cast<uint8_t*>(const_cast<void*>(v));
  p.pool.ks = const_cast<float*>(ks);
  p.pool.vs = const_cast<float*>(vs);
  p.width = c->table_width;
  p.table = table;
  p.past = past;
  p.counts = counts;
  return p;
}

}  // namespace

extern "C" {

int lc_rotary_turns(int32_t pairs, const double* inv_freq, uint64_t* turns) {
  if (pairs <= 0) return set_error(LC_ERR_INVALID, "pairs must be positive");
  if (!inv_freq || !turns) return set_error(LC_ERR_INVALID, "null pointer argument");
  for (int32_t i = 0; i < pairs; ++i)
    if (!std::isfinite(inv_freq[i])) return set_error(LC_ERR_INVALID, "frequencies must be finite");
  for (int32_t i = 0; i < pairs; ++i) {
    // 64 significant bits (x87); whole turns do not matter.
    long double t = (long double)inv_freq[i] / 6.283185307179586476925286766559005768L;
    t -= std::floor(t);
    const long double u = std::nearbyint(std::ldexp(t, 64));
    turns[i] = u >= 18446744073709551616.0L ? 0 : (uint64_t)u;
  }
  return LC_OK;
}

int lc_rotary_apply(const lc_rotary_t* rotary, int32_t dtype, int64_t batch, int64_t tokens,
                    int32_t heads, const int64_t* positions, int64_t pos0, int32_t inverse,
                    const void* x, const lc_rows_t* x_rows, void* out, const lc_rows_t* out_rows,
                    void* stream) {
  if (int rc = check_rotary(rotary)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (batch < 0 || tokens < 0 || heads <= 0)
    return set_error(LC_ERR_INVALID, "rotary positions need batch, tokens >= 0 and heads > 0");
  if (inverse != 0 && inverse != 1) return set_error(LC_ERR_INVALID, "inverse must be 0 or 1");
  if (batch == 0 || tokens == 0) return LC_OK;
  if (batch > 1 << 24 || tokens > 1 << 24 || heads > 1 << 16 || batch * tokens > kMostGroups ||
      batch * tokens * heads > (int64_t)1 << 32)
    return set_error(LC_ERR_UNSUPPORTED, "the rows exceed the kernels' grids");
  if (!x || !out) return set_error(LC_ERR_INVALID, "null pointer argument");
  if (!aligned(positions, 8)) return set_error(LC_ERR_INVALID, "positions must be 8-byte aligned");
  const size_t e = dtype == LC_DTYPE_BF16 ? 2 : 4;
  if (!aligned(x, e) || !aligned(out, e))
    return set_error(LC_ERR_INVALID, "x and out must be aligned to their elements");
  const Rows xr{batch, tokens, heads, rotary->head_dim, x_rows, e};
  const Rows orr{batch, tokens, heads, rotary->head_dim, out_rows, e};
  if (int rc = xr.check("x")) return rc;
  if (int rc = orr.check("out")) return rc;
  if (int rc = orr.check_written("out")) return rc;
  const bool in_place = x == out && xr.same(orr);
  if (!in_place && meet(xr.bytes(x), orr.bytes(out)))
    return set_error(LC_ERR_INVALID, "out must be x or not overlap it");
  const Range w = orr.bytes(out);
  if (meet(w, range(positions, (size_t)(batch * tokens) * 8)) ||
      meet(w, range(rotary->turns, (size_t)rotary->rotary_dim * 4)))
    return set_error(LC_ERR_INVALID, "out must not overlap positions or turns");
  lc::RotaryProblem p;
  p.dtype = dtype;
  p.batch = batch;
  p.tokens = tokens;
  p.heads = heads;
  p.D = rotary->head_dim;
  p.turns = make_turns(rotary);
  p.inverse = inverse != 0;
  p.positions = positions;
  p.pos0 = pos0;
  p.x = x;
  p.out = out;
  p.xs = head_rows(x_rows);
  p.os = head_rows(out_rows);
  p.align = (int)e;
  for (int bytes : {8, 16})
    if (xr.vec(x, bytes) && orr.vec(out, bytes)) p.align = bytes;
  p.copy = !in_place;
  hipError_t err = lc::launch_rotary(p, static_cast<hipStream_t>(stream));
  return err == hipSuccess ? LC_OK : hip_error(err, "lc_rotary_apply launch");
}

int lc_paged_append(const lc_paged_t* cache, const lc_rotary_t* rotary, const int32_t* table,
                    const int32_t* past, const int32_t* counts, const void* q,
                    const lc_rows_t* q_rows, void* q_out, const void* k, const lc_rows_t* k_rows,
                    const void* v, const lc_rows_t* v_rows, void* k_pages, void* v_pages,
                    float* k_scales, float* v_scales, void* stream) {
  if (int rc = check_paged(cache, q != nullptr)) return rc;
  if (rotary) {
    if (int rc = check_rotary(rotary)) return rc;
    if (rotary->head_dim != cache->head_dim)
      return set_error(LC_ERR_INVALID, "rotary and the cache must agree in head_dim");
    if (rotary->rotary_dim % 16 != 0)
      return set_error(LC_ERR_UNSUPPORTED, "the append needs rotary_dim %% 16 == 0");
  }
  if (cache->tokens == 0) return LC_OK;
  if (!k || !v) return set_error(LC_ERR_INVALID, "null pointer argument");
  if ((q != nullptr) != (q_out != nullptr)) return set_error(LC_ERR_INVALID, "q and q_out come together");
  if (q && !rotary) return set_error(LC_ERR_INVALID, "queries are given to be rotated");
  PoolRanges pool;
  if (int rc = check_pool(cache, table, past, counts, k_pages, v_pages, k_scales, v_scales, &pool)) return rc;
  const size_t e = cache->dtype == LC_DTYPE_BF16 ? 2 : 4;
  if (!aligned(k, e) || !aligned(v, e) || !aligned(q, e) || !aligned(q_out, e))
    return set_error(LC_ERR_INVALID, "q, k, v and q_out must be aligned to their elements");
  const int64_t B = cache->batch, N = cache->tokens, D = cache->head_dim;
  const lc_rows_t dense = {N * cache->heads_q * D, cache->heads_q * D, D};
  const Rows qr{B, N, cache->heads_q, D, q_rows, e}, kr{B, N, cache->heads_kv, D, k_rows, e},
      vr{B, N, cache->heads_kv, D, v_rows, e}, outr{B, N, cache->heads_q, D, &dense, e};
  if (int rc = kr.check("k")) return rc;
  if (int rc = vr.check("v")) return rc;
  if (q)
    if (int rc = qr.check("q")) return rc;
  Range ins[6] = {kr.bytes(k), vr.bytes(v), q ? qr.bytes(q) : Range{0, 0}, pool.r[4], pool.r[5], pool.r[6]};
  for (const Range& i : ins)
    for (int o = 0; o < 4; ++o)
      if (meet(i, pool.r[o]))
        return set_error(LC_ERR_INVALID, "pages and scales must not overlap the inputs");
  if (rotary)
    for (int o = 0; o < 4; ++o)
      if (meet(range(rotary->turns, (size_t)rotary->rotary_dim * 4), pool.r[o]))
        return set_error(LC_ERR_INVALID, "pages and scales must not overlap the inputs");
  if (q) {
    const Range w = outr.bytes(q_out);
    const bool in_place = q == q_out && qr.same(outr);
    for (int i = 0; i < 6; ++i)
      if (!(i == 2 && in_place) && meet(w, ins[i]))
        return set_error(LC_ERR_INVALID, "q_out must be q or not overlap the inputs");
    for (int o = 0; o < 4; ++o)
      if (meet(w, pool.r[o])) return set_error(LC_ERR_INVALID, "q_out must not overlap pages or scales");
    if (meet(w, range(rotary->turns, (size_t)rotary->rotary_dim * 4)))
      return set_error(LC_ERR_INVALID, "q_out must be q or not overlap the inputs");
  }
  const int64_t touched = (N + cache->page_rows - 2) / cache->page_rows + 1;
  if (B * touched * cache->heads_kv * 2 + B * N > kMostGroups)
    return set_error(LC_ERR_UNSUPPORTED, "the cache or its tokens exceed the kernels' grids");
  lc::AppendProblem p;
  p.p = make_problem(cache, table, past, counts, k_pages, v_pages, k_scales, v_scales);
  p.turns = make_turns(rotary);
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_out = q_out;
  p.qs = q ? head_rows(q_rows) : lc::HeadRows{0, 0, 0};
  p.ks = head_rows(k_rows);
  p.vs = head_rows(v_rows);
  p.vec = kr.vec(k) && vr.vec(v) && (!q || (qr.vec(q) && outr.vec(q_out)));
  hipError_t err = lc::launch_paged_append(p, static_cast<hipStream_t>(stream));
  return err == hipSuccess ? LC_OK : hip_error(err, "lc_paged_append launch");
}

size_t lc_paged_attn_workspace_bytes(const lc_paged_t* cache) {
  if (check_paged(cache, true) || cache->tokens == 0) return 0;
  return lc::paged_attn_bytes(make_problem(cache, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr));
}

int lc_paged_attn(const lc_paged_t* cache, const int32_t* table, const int32_t* past,
                  const int32_t* counts, const void* q, const void* k_pages, const void* v_pages,
                  const float* k_scales, const float* v_scales, void* out, float* m, float* l,
                  void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_paged(cache, true)) return rc;
  if (cache->tokens == 0) return LC_OK;
  if (!q || !out) return set_error(LC_ERR_INVALID, "null pointer argument");
  PoolRanges pool;
  if (int rc = check_pool(cache, table, past, counts, k_pages, v_pages, k_scales, v_scales, &pool)) return rc;
  if (!aligned(q, 16) || !aligned(out, 16)) return set_error(LC_ERR_INVALID, "q and out must be 16-byte aligned");
  if (!aligned(m, 4) || !aligned(l, 4)) return set_error(LC_ERR_INVALID, "m and l must be 4-byte aligned");
  const lc::PagedProblem p = make_problem(cache, table, past, counts, k_pages, v_pages, k_scales, v_scales);
  const size_t need = lc::paged_attn_bytes(p);
  if (workspace_bytes < need || (need && !workspace))
    return set_error(LC_ERR_WORKSPACE, "paged attention needs a workspace of %zu bytes, got %zu", need,
                     workspace ? workspace_bytes : (size_t)0);
  if (!aligned(workspace, 16))
    return set_error(LC_ERR_INVALID, "the workspace must be 16-byte aligned");
  const size_t rows = (size_t)cache->batch * cache->tokens * cache->heads_q;
  const size_t e = cache->dtype == LC_DTYPE_BF16 ? 2 : 4;
  const Range io[5] = {range(out, rows * cache->head_dim * e), range(m, rows * 4), range(l, rows * 4),
                       range(workspace, need), range(q, rows * cache->head_dim * e)};
  for (int i = 0; i < 5; ++i)
    for (int j = i + 1; j < 5; ++j)
      if (meet(io[i], io[j]))
        return set_error(LC_ERR_INVALID, "q, out, m, l and the workspace must not overlap each other");
  for (int i = 0; i < 4; ++i)
    for (const Range& r : pool.r)
      if (meet(io[i], r)) return set_error(LC_ERR_INVALID, "outputs must not overlap the cache or its lengths");
  hipError_t err = lc::launch_paged_attn(p, q, out, m, l, workspace, static_cast<hipStream_t>(stream));
  return err == hipSuccess ? LC_OK : hip_error(err, "lc_paged_attn launch");
}

}  // extern "C"
