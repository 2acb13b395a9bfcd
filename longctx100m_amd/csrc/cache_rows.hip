// Rows of a KV cache that go and rows that move (gfx950): eviction by
// accumulated weight, and the commit of an accepted path of drafted tokens.
//
// Eviction of a head's L rows to a budget of n: rows are ranked by (protected,
// weight), ties by the lower row.  Each row's rank is a 32-bit key that orders
// as the weights do, so the smallest kept key T and the number of rows with
// that very key that stay come from three histogram passes over the key's
// digits (11, 11 and 10 bits).  The kept rows below n stay where they are; the
// others, ascending, go to the holes below n, ascending.  Sources lie at n and
// above and targets below, so all moves run at once and in place, and no row
// moves that could stay: a cache that is cut back by a few rows costs a few
// rows' copies.
#include "common.h"
#include "cache.h"

#include <algorithm>

namespace lc {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 16;                    // consecutive rows of a thread
constexpr int kChunk = kThreads * kPer;     // rows of a workgroup
constexpr int kDigits = 3;
constexpr int kBins = 2048;
__host__ __device__ constexpr int shift_of(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }

struct EvictArgs {
  int B, C, Hkv, budget, sinks, recent;
  int chunks_a, chunks;  // chunks of rows below the budget, and of all rows
  const int32_t *lens, *kept, *ends;
  const float* w;
  const int32_t* pos;
  float* w_out;
  int32_t *pos_out, *lens_out;
  // Workspace, per (sequence, head): histograms, the chunks' (above, equal)
  // counts, holes and movers, the number of moves.
  uint32_t* hist;
  int2* counts;
  int32_t *holes, *movers, *moves;
  int half;  // room of holes and movers
};

struct RowInfo {
  int b, L, kept, end;
};
__device__ __forceinline__ RowInfo row_info(const EvictArgs& a, int bh) {
  RowInfo r;
  r.b = bh / a.Hkv;
  r.L = max(0, min(a.lens[r.b], a.C));
  r.kept = a.kept ? min(a.kept[r.b], r.L) : 0;
  r.end = a.ends ? a.ends[r.b] : r.L;
  return r;
}
__device__ __forceinline__ int position(const EvictArgs& a, const RowInfo& r, int64_t base, int j) {
  return j < r.kept ? a.pos[base + j] : (int)((int64_t)r.end - r.L + j);
}
// The rank of row j: larger stays longer.
__device__ __forceinline__ uint32_t rank_key(const EvictArgs& a, const RowInfo& r, int64_t base,
                                             int j) {
  const int p = position(a, r, base, j);
  if (p < a.sinks || (int64_t)p >= (int64_t)r.end - a.recent) return 0xffffffffu;
  const float w = a.w[base + j];
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 counts as 0
  return u >> 31 ? ~u : u | 0x80000000u;
}

// Rows of a chunk: those below the budget and those from it on lie in
// different chunks.
struct Chunk {
  int lo, hi;
};
__device__ __forceinline__ Chunk chunk_of(const EvictArgs& a, int x, int L) {
  Chunk c;
  const int n = min(a.budget, L);
  if (x < a.chunks_a) {
    c.lo = min(x * kChunk, n);
    c.hi = min(c.lo + kChunk, n);
  } else {
    c.lo = (int)min((int64_t)a.budget + (int64_t)(x - a.chunks_a) * kChunk, (int64_t)L);
    c.hi = (int)min((int64_t)c.lo + kChunk, (int64_t)L);
  }
  return c;
}

// Exclusive prefix sum of x over the workgroup, and the sum of all.
__device__ __forceinline__ int2 block_scan(int x, int* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int inc = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(inc, off, 64);
    if (lane >= off) inc += y;
  }
  __syncthreads();  // part may still be in use
  if (lane == 63) part[wave] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) before += part[w];
    all += part[w];
  }
  return make_int2(before + inc - x, all);
}

// The digits of the smallest kept key found so far, and how many of the rows
// that share them stay.
struct Cut {
  uint32_t prefix;
  int need;
};
// From the histograms of the passes before `passes`; by the whole workgroup.
__device__ __forceinline__ Cut find_cut(const EvictArgs& a, int bh, int passes, int* part, int* pick) {
  Cut cut{0u, a.budget};
  for (int p = 0; p < passes; ++p) {
    const uint32_t* h = a.hist + ((int64_t)bh * kDigits + p) * kBins;
    // Bins from the top: thread t holds 8 of them, the largest first.
    int cnt[kBins / kThreads], sum = 0;
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) {
      cnt[i] = (int)h[kBins - 1 - (threadIdx.x * (kBins / kThreads) + i)];
      sum += cnt[i];
    }
    int above = block_scan(sum, part).x;
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) {
      if (above < cut.need && above + cnt[i] >= cut.need) {
        pick[0] = kBins - 1 - (threadIdx.x * (kBins / kThreads) + i);
        pick[1] = cut.need - above;
      }
      above += cnt[i];
    }
    __syncthreads();
    cut.prefix |= (uint32_t)pick[0] << shift_of(p);
    cut.need = pick[1];
    __syncthreads();
  }
  return cut;
}

__global__ __launch_bounds__(kThreads) void evict_clear_kernel(uint32_t* hist, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i < n) hist[i] = 0;
}

// Histogram of digit `pass` of the keys that share the digits before it.
__global__ __launch_bounds__(kThreads) void evict_hist_kernel(EvictArgs a, int pass) {
  __shared__ uint32_t h[kBins];
  __shared__ int part[kThreads / 64], pick[2];
  const int bh = blockIdx.x / a.chunks, x = blockIdx.x - bh * a.chunks;
  const RowInfo r = row_info(a, bh);
  const Chunk c = chunk_of(a, x, r.L);
  if (r.L <= a.budget || c.lo >= c.hi) return;
  for (int i = threadIdx.x; i < kBins; i += kThreads) h[i] = 0;
  const Cut cut = find_cut(a, bh, pass, part, pick);
  __syncthreads();
  const int64_t base = (int64_t)bh * a.C;
  const int sh = shift_of(pass);
  const uint32_t mask = pass == 0 ? 0u : ~0u << shift_of(pass - 1);
  const uint32_t digit = pass == 2 ? 1023u : 2047u;
  for (int j = c.lo + threadIdx.x; j < c.hi; j += kThreads) {
    const uint32_t k = rank_key(a, r, base, j);
    if ((k & mask) == cut.prefix) atomicAdd(&h[k >> sh & digit], 1u);
  }
  __syncthreads();
  uint32_t* out = a.hist + ((int64_t)bh * kDigits + pass) * kBins;
  for (int i = threadIdx.x; i < kBins; i += kThreads)
    if (h[i]) atomicAdd(&out[i], h[i]);  // whole numbers: the order does not matter
}

// How many of a chunk's rows rank above the smallest kept key, and how many have it.
__global__ __launch_bounds__(kThreads) void evict_count_kernel(EvictArgs a) {
  __shared__ int part[kThreads / 64], pick[2];
  const int bh = blockIdx.x / a.chunks, x = blockIdx.x - bh * a.chunks;
  const RowInfo r = row_info(a, bh);
  if (r.L <= a.budget) return;
  const Chunk c = chunk_of(a, x, r.L);
  const Cut cut = find_cut(a, bh, kDigits, part, pick);
  const int64_t base = (int64_t)bh * a.C;
  int gt = 0, eq = 0;
  for (int j = c.lo + threadIdx.x; j < c.hi; j += kThreads) {
    const uint32_t k = rank_key(a, r, base, j);
    gt += k > cut.prefix;
    eq += k == cut.prefix;
  }
  const int gts = block_scan(gt, part).y, eqs = block_scan(eq, part).y;
  if (threadIdx.x == 0) a.counts[(int64_t)bh * a.chunks + x] = make_int2(gts, eqs);
}

// Which rows of a chunk stay, and the holes or movers among them.
__global__ __launch_bounds__(kThreads) void evict_plan_kernel(EvictArgs a) {
  __shared__ int part[kThreads / 64], pick[2];
  const int bh = blockIdx.x / a.chunks, x = blockIdx.x - bh * a.chunks;
  const RowInfo r = row_info(a, bh);
  const Chunk c = chunk_of(a, x, r.L);
  const int64_t base = (int64_t)bh * a.C;
  const bool lower = x < a.chunks_a;
  if (x == 0 && bh % a.Hkv == 0 && threadIdx.x == 0) a.lens_out[r.b] = min(r.L, a.budget);
  const int first = c.lo + threadIdx.x * kPer;  // the thread's rows, in order
  if (r.L <= a.budget) {
    for (int j = c.lo + threadIdx.x; j < c.hi; j += kThreads) {
      a.w_out[base + j] = a.w[base + j];
      a.pos_out[base + j] = position(a, r, base, j);
    }
    if (x == 0 && threadIdx.x == 0) a.moves[bh] = 0;
    return;
  }
  const Cut cut = find_cut(a, bh, kDigits, part, pick);
  // Over the chunks before this one: rows with the smallest kept key, then
  // (with how many of those stay) the holes or movers.
  int eq_before = 0;
  for (int i0 = 0; i0 < a.chunks; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    eq_before += block_scan(i < x ? a.counts[(int64_t)bh * a.chunks + i].y : 0, part).y;
  }
  int before = 0, all = 0, eq_run = 0;
  for (int i0 = 0; i0 < a.chunks; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    const int2 n = i < a.chunks ? a.counts[(int64_t)bh * a.chunks + i] : make_int2(0, 0);
    const int2 e = block_scan(n.y, part);
    const int stay = n.x + min(max(cut.need - eq_run - e.x, 0), n.y);
    eq_run += e.y;
    int cnt = 0;
    if (i < a.chunks && (i < a.chunks_a) == lower) {
      const Chunk ci = chunk_of(a, i, r.L);
      cnt = lower ? ci.hi - ci.lo - stay : stay;
    }
    before += block_scan(i < x ? cnt : 0, part).y;
    all += block_scan(cnt, part).y;
  }
  if (x == 0 && threadIdx.x == 0) a.moves[bh] = all;  // holes
  uint32_t key[kPer];
  int eq = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    key[i] = first + i < c.hi ? rank_key(a, r, base, first + i) : 0u;
    eq += first + i < c.hi && key[i] == cut.prefix;
  }
  int left = cut.need - eq_before - block_scan(eq, part).x;  // equal rows that still stay
  uint32_t keep = 0;
  int listed = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (first + i >= c.hi) continue;
    const bool same = key[i] == cut.prefix;
    const bool k = key[i] > cut.prefix || (same && left > 0);
    left -= same;
    keep |= (uint32_t)k << i;
    listed += k != lower;
  }
  int at = before + block_scan(listed, part).x;
  int32_t* list = (lower ? a.holes : a.movers) + (int64_t)bh * a.half;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int j = first + i;
    if (j >= c.hi) continue;
    const bool k = keep >> i & 1;
    if (k != lower) list[at++] = j;
    if (k && lower) {
      a.w_out[base + j] = a.w[base + j];
      a.pos_out[base + j] = position(a, r, base, j);
    }
  }
}

struct MoveArgs {
  uint8_t *k, *v;
  int64_t seq, row, head;  // bytes
  int chunks;              // 16-byte chunks of a row of one head
  int blocks;              // workgroups of a (sequence, head)
};

// Thread: one 16-byte chunk of K and V of a move.
__global__ __launch_bounds__(kThreads) void evict_move_kernel(EvictArgs a, MoveArgs t) {
  const int bh = blockIdx.x / t.blocks, x = blockIdx.x - bh * t.blocks;
  const int n = a.moves[bh];
  if (n == 0) return;
  const RowInfo r = row_info(a, bh);
  const int64_t base = (int64_t)bh * a.C;
  const int64_t off = r.b * t.seq + (bh % a.Hkv) * t.head;
  const int64_t total = (int64_t)n * t.chunks;
  for (int64_t i = (int64_t)x * kThreads + threadIdx.x; i < total; i += (int64_t)t.blocks * kThreads) {
    const int mv = (int)(i / t.chunks), ch = (int)(i - (int64_t)mv * t.chunks);
    const int dst = a.holes[(int64_t)bh * a.half + mv], src = a.movers[(int64_t)bh * a.half + mv];
    const int64_t so = off + src * t.row + 16 * ch, d = off + dst * t.row + 16 * ch;
    const uint4 kx = *reinterpret_cast<const uint4*>(t.k + so);
    const uint4 vx = *reinterpret_cast<const uint4*>(t.v + so);
    *reinterpret_cast<uint4*>(t.k + d) = kx;
    *reinterpret_cast<uint4*>(t.v + d) = vx;
    if (ch == 0) {
      a.w_out[base + dst] = a.w[base + src];
      a.pos_out[base + dst] = position(a, r, base, src);
    }
  }
}

// Thread: one 16-byte chunk of every row of a path, in the order of the path.
// A row's target is never above its source and sources ascend, so eight rows
// are read before the first of them is written.
__global__ __launch_bounds__(256) void cache_commit_kernel(CommitArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = a.Hkv * a.chunks;
  const int b = (int)(i / per);
  if (b >= a.B) return;
  const int hc = (int)(i - (int64_t)b * per);
  const int h = hc / a.chunks, ch = hc - h * a.chunks;
  const int past = a.past[b];
  uint8_t* base = (blockIdx.z ? a.v : a.k)[blockIdx.y];
  const bool moves = base != nullptr;
  base += b * a.seq + h * a.head + 16 * ch + past * a.row;
  const int room = past < 0 ? 0 : (int)max((int64_t)0, (int64_t)a.C - past);
  const int32_t* path = a.path + (int64_t)b * a.P;
  int last = -1, n = 0;
  bool on = true;
  for (int j0 = 0; j0 < a.P && on; j0 += 8) {
    uint4 x[8];
    int src[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int p = j0 + e < a.P ? path[j0 + e] : -1;
      on = on && p > last && p < room;
      src[e] = on ? p : -1;
      if (on) {
        last = p;
        ++n;
        if (moves && p != j0 + e) x[e] = *reinterpret_cast<const uint4*>(base + p * a.row);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (moves && src[e] >= 0 && src[e] != j0 + e)
        *reinterpret_cast<uint4*>(base + (j0 + e) * a.row) = x[e];
  }
  if (a.lens_out && hc == 0 && blockIdx.y == 0 && blockIdx.z == 0)
    a.lens_out[b] = past < 0 ? past : past + n;
}

struct Layout {
  int chunks_max, half;
  size_t hist, counts, list, moves, total;
};
Layout layout_of(int B, int Hkv, int C) {
  Layout y;
  const size_t bh = (size_t)B * Hkv;
  y.chunks_max = (C + kChunk - 1) / kChunk + 1;  // whatever the budget
  y.half = C / 2 + 1;                            // moves: at most min(budget, C - budget)
  y.hist = bh * kDigits * kBins * 4;
  y.counts = (bh * y.chunks_max * 8 + 15) / 16 * 16;
  y.list = (bh * y.half * 4 + 15) / 16 * 16;
  y.moves = (bh * 4 + 15) / 16 * 16;
  y.total = y.hist + y.counts + 2 * y.list + y.moves;
  return y;
}

}  // namespace

size_t cache_evict_bytes(int B, int Hkv, int C) { return layout_of(B, Hkv, C).total; }

hipError_t launch_cache_evict(const EvictProblem& p, void* ws, hipStream_t s) {
  const Layout y = layout_of(p.B, p.Hkv, p.C);
  const int bh = p.B * p.Hkv;
  EvictArgs a;
  a.B = p.B;
  a.C = p.C;
  a.Hkv = p.Hkv;
  a.budget = p.budget;
  a.sinks = p.sinks;
  a.recent = p.recent;
  a.chunks_a = (p.budget + kChunk - 1) / kChunk;
  a.chunks = a.chunks_a + (p.C - p.budget + kChunk - 1) / kChunk;
  a.lens = p.lens;
  a.kept = p.kept;
  a.ends = p.ends;
  a.w = p.w;
  a.pos = p.pos;
  a.w_out = p.w_out;
  a.pos_out = p.pos_out;
  a.lens_out = p.lens_out;
  uint8_t* at = static_cast<uint8_t*>(ws);
  a.hist = reinterpret_cast<uint32_t*>(at);
  a.counts = reinterpret_cast<int2*>(at += y.hist);
  a.holes = reinterpret_cast<int32_t*>(at += y.counts);
  a.movers = reinterpret_cast<int32_t*>(at += y.list);
  a.moves = reinterpret_cast<int32_t*>(at += y.list);
  a.half = y.half;
  const dim3 grid((unsigned)(bh * a.chunks)), block(kThreads);
  if (p.C > p.budget) {
    const int64_t n = (int64_t)bh * kDigits * kBins;
    hipLaunchKernelGGL(evict_clear_kernel, dim3((unsigned)((n + kThreads - 1) / kThreads)), block, 0, s,
                       a.hist, n);
    for (int pass = 0; pass < kDigits; ++pass)
      hipLaunchKernelGGL(evict_hist_kernel, grid, block, 0, s, a, pass);
    hipLaunchKernelGGL(evict_count_kernel, grid, block, 0, s, a);
  }
  hipLaunchKernelGGL(evict_plan_kernel, grid, block, 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.C <= p.budget) return e;
  MoveArgs t;
  t.k = static_cast<uint8_t*>(p.k);
  t.v = static_cast<uint8_t*>(p.v);
  t.seq = p.seq * p.elem;
  t.row = p.row * p.elem;
  t.head = p.head * p.elem;
  t.chunks = p.D * p.elem / 16;
  const int64_t most = (int64_t)std::min(p.budget, p.C - p.budget) * t.chunks;
  t.blocks = (int)std::max<int64_t>(1, std::min<int64_t>((most + kThreads - 1) / kThreads, std::max(1, 2048 / bh)));
  hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)(bh * t.blocks)), block, 0, s, a, t);
  return hipGetLastError();
}

hipError_t launch_cache_commit(const CommitArgs& a, int layers, hipStream_t s) {
  const int64_t threads = (int64_t)a.B * a.Hkv * a.chunks;
  const dim3 grid((unsigned)((threads + 255) / 256), (unsigned)std::max(1, layers), layers > 0 ? 2 : 1);
  hipLaunchKernelGGL(cache_commit_kernel, grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace lc
