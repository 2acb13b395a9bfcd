// Rows of a KV cache that go and rows that move (gfx950): eviction by
// accumulated weight, and the commit of an accepted path of drafted tokens.
//
// Eviction of a head's L rows to a budget of n: rows are ranked by (protected,
// weight), ties by the lower row.  Each row's rank is a 32-bit key that orders
// as the weights do, so the smallest kept key and the number of rows with that
// very key that stay (the cut) come from three histograms over the key's digits
// (11, 11 and 10 bits).  The kept rows below n stay where they are; the
// others, ascending, go to the holes below n, ascending.  Sources lie at n and
// above and targets below, so all moves run at once and in place, and no row
// moves that could stay: a cache that is cut back by a few rows costs a few
// rows' copies.
//
// Up to kShortRows rows one workgroup holds a head's keys in registers and plans
// it in one launch.  Longer heads are split over the chip, one launch for each
// histogram (a digit needs all of the digits before it) and one that plans.
// Every chunk leaves its histogram by itself and the next launch adds them up:
// adding them in memory costs more (64 chunks' atomics to the same bins from
// all XCDs: 10 us a launch), and needs a cleared array.  What is left is a few
// microseconds of latency and instructions a launch, so a thread loads its
// consecutive rows in vectors, all before the first is used.
#include "common.h"
#include "cache.h"

#include <algorithm>

namespace lc {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kPer = 16;                // rows of a thread of the long form
constexpr int kThreads = 512;           // of a workgroup of it
constexpr int kPart = kThreads * kPer;  // rows that it holds at a time
constexpr int kParts = 7;               // at most: a chunk's histogram has 16-bit bins
// Capacity of the short form: at most 16,000 rows of eight heads take it 21 us where
// the long form's launches take 34, 4,000 11 against 31.  (The lengths are not
// known on the host: 4,000 rows in a capacity of 32,768 take the 32 of the long
// form, in one of 262,144 46.)
constexpr int kShortRows = 1024 * 16;
// Chunks (of K and V, 16 bytes each) up to which the planning workgroup of the
// short form moves them itself, which saves a launch: 100 of 4,300 rows of 256
// bytes 12.1 us against 14.5, but 500 of 4,000 22 against 13.6.
constexpr int kFewMoves = 4096;
constexpr int kDigits = 3;
constexpr int kBins = 2048;
__host__ __device__ constexpr int shift_of(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__host__ __device__ constexpr uint32_t digit_mask(int pass) { return pass == 2 ? 1023u : 2047u; }
// The bits of the digits before a pass.
__host__ __device__ constexpr uint32_t prefix_mask(int pass) {
  return pass == 0 ? 0u : ~0u << shift_of(pass - 1);
}

// The digits of the smallest kept key found so far, and how many of the rows
// that share them stay.
struct Cut {
  uint32_t prefix;
  int need;
};

struct EvictArgs {
  int B, C, Hkv, budget, sinks, recent;
  int chunk;             // rows of a workgroup of the long form, a multiple of kPart
  int chunks_a, chunks;  // chunks of rows below the budget, and of all rows
  const int32_t *lens, *kept, *ends;
  const float* w;
  const int32_t* pos;
  float* w_out;
  int32_t *pos_out, *lens_out;
  // Workspace, per (sequence, head): the chunks' histograms of each pass, the
  // cuts, the chunks' rows above the last pass's prefix, holes and movers, the
  // number of moves.
  uint16_t* hist;  // [pass][head][chunk][bin]
  Cut* cuts;
  int32_t *above, *holes, *movers, *moves;
  int half;  // room of holes and movers
};

struct RowInfo {
  int b, L, kept, end;
  int recent_from;  // positions from here on are protected
};
__device__ __forceinline__ RowInfo row_info(const EvictArgs& a, int bh) {
  RowInfo r;
  r.b = bh / a.Hkv;
  r.L = max(0, min(a.lens[r.b], a.C));
  r.kept = a.kept ? min(a.kept[r.b], r.L) : 0;
  r.end = a.ends ? a.ends[r.b] : r.L;
  r.recent_from = (int)max((int64_t)r.end - a.recent, (int64_t)INT32_MIN);
  return r;
}
__device__ __forceinline__ int position(const EvictArgs& a, const RowInfo& r, int64_t base, int j) {
  return j < r.kept ? a.pos[base + j] : (int)((int64_t)r.end - r.L + j);
}
// A key that orders as the weights do (-0 as 0), NaN below all.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  const uint32_t k = u ^ (uint32_t)((int32_t)u >> 31 | (int32_t)0x80000000);
  return w != w ? 0u : k;
}
constexpr uint32_t kProtected = 0xffffffffu;

// The weights, positions and keys of a thread's P rows from `first` on, n of
// them below row hi (keys past them: 0).
template <int P>
struct Rows {
  float w[P];
  int pos[P];
  uint32_t key[P];
  int n;
};
template <int P>
__device__ __forceinline__ void load_rows(const EvictArgs& a, const RowInfo& r, int64_t base, int first,
                                          int hi, Rows<P>& x) {
  x.n = max(0, min(hi - first, P));
  if (x.n == P) {
    const float* p = a.w + base + first;
#pragma unroll
    for (int i = 0; i < P; i += 4) {
      const f32x4u v = *reinterpret_cast<const f32x4u*>(p + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) x.w[i + e] = v[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) x.w[i] = i < x.n ? a.w[base + first + i] : 0.f;
  }
  const int p0 = (int)((int64_t)r.end - r.L + first);
#pragma unroll
  for (int i = 0; i < P; ++i) x.pos[i] = p0 + i;
  if (x.n > 0 && first < r.kept) {
    int old[P];
#pragma unroll
    for (int i = 0; i < P; ++i) old[i] = a.pos[base + min(first + i, r.kept - 1)];
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (first + i < r.kept) x.pos[i] = old[i];
  }
#pragma unroll
  for (int i = 0; i < P; ++i) x.key[i] = weight_key(x.w[i]);
  if (first < r.kept || p0 < a.sinks || (int64_t)p0 + P > r.recent_from) {  // elsewhere none is protected
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (x.pos[i] < a.sinks || x.pos[i] >= r.recent_from) x.key[i] = kProtected;
  }
  if (x.n < P) {
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (i >= x.n) x.key[i] = 0u;
  }
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
    c.lo = (int)min((int64_t)x * a.chunk, (int64_t)n);
    c.hi = (int)min((int64_t)c.lo + a.chunk, (int64_t)n);
  } else {
    c.lo = (int)min((int64_t)a.budget + (int64_t)(x - a.chunks_a) * a.chunk, (int64_t)L);
    c.hi = (int)min((int64_t)c.lo + a.chunk, (int64_t)L);
  }
  return c;
}

// Exclusive prefix sums of x over a workgroup of NT threads, and the sum.
struct Scan {
  int before, all;
};
template <int NT>
__device__ __forceinline__ Scan block_scan(int x, int* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int inc = wave_scan(x);
  __syncthreads();  // part may still be in use
  if (lane == 63) part[wave] = inc;
  __syncthreads();
  Scan s{inc - x, 0};
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    const int y = part[w];
    if (w < wave) s.before += y;
    s.all += y;
  }
  return s;
}

// Adds the digits of a thread's keys that share the prefix to the histogram h
// (in LDS); keys that agree (many equal weights) are added at once.
template <int P>
__device__ __forceinline__ void count_digits(const Rows<P>& x, uint32_t prefix, int pass, uint32_t* h) {
  if (x.n == 0) return;
  const uint32_t mask = prefix_mask(pass);
  uint32_t diff = 0;
#pragma unroll
  for (int i = 1; i < P; ++i)
    if (i < x.n) diff |= x.key[i] ^ x.key[0];
  if (diff >> shift_of(pass) == 0) {
    if ((x.key[0] & mask) == prefix)
      atomicAdd(&h[x.key[0] >> shift_of(pass) & digit_mask(pass)], (uint32_t)x.n);
    return;
  }
#pragma unroll
  for (int i = 0; i < P; ++i)
    if (i < x.n && (x.key[i] & mask) == prefix)
      atomicAdd(&h[x.key[i] >> shift_of(pass) & digit_mask(pass)], 1u);
}

// The bin that the cut falls into; by the whole workgroup, thread t with the
// counts of bins kBins - 1 - t * kOwn - i.  need: rows that stay of those
// counted (1 .. their number).
template <int NT>
__device__ __forceinline__ Cut narrow(Cut cut, const int (&cnt)[kBins / NT], int pass, int* part,
                                      int* pick) {
  constexpr int kOwn = kBins / NT;
  int sum = 0;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) sum += cnt[i];
  int over = block_scan<NT>(sum, part).before;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    if (over < cut.need && over + cnt[i] >= cut.need) {
      pick[0] = kBins - 1 - (threadIdx.x * kOwn + i);
      pick[1] = cut.need - over;
    }
    over += cnt[i];
  }
  __syncthreads();
  cut.prefix |= (uint32_t)pick[0] << shift_of(pass);
  cut.need = pick[1];
  return cut;
}

// Which of a thread's rows stay.  left: of the rows with the cut's own key, how
// many still stay from its first row on.
template <int P>
__device__ __forceinline__ uint32_t staying(const Rows<P>& x, uint32_t cut, int left) {
  uint32_t keep = 0;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (i >= x.n) continue;
    const bool same = x.key[i] == cut;
    keep |= (uint32_t)(x.key[i] > cut || (same && left > 0)) << i;
    left -= same;
  }
  return keep;
}
template <int P>
__device__ __forceinline__ int equal_rows(const Rows<P>& x, uint32_t cut) {
  int eq = 0;
#pragma unroll
  for (int i = 0; i < P; ++i) eq += i < x.n && x.key[i] == cut;
  return eq;
}

// Writes the weights and positions of the rows from lo on, below hi, whose bit
// is set in keep (in LDS, P rows a word): consecutive lanes, consecutive rows
// (thread by thread the 2 x 16 stores of a wave touch 64 lines each: 8 us).
// Inputs may be the outputs: a thread reads all its rows first.
template <int P, int NT>
__device__ __forceinline__ void write_kept(const EvictArgs& a, const RowInfo& r, int64_t base, int lo,
                                           int hi, const uint32_t* keep) {
  float w[P];
  int p[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int j = min(lo + (int)threadIdx.x + i * NT, hi - 1);
    w[i] = a.w[base + j];
    p[i] = position(a, r, base, j);
  }
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int x = threadIdx.x + i * NT;
    if (lo + x >= hi || !(keep[x / P] >> (x % P) & 1)) continue;
    a.w_out[base + lo + x] = w[i];
    a.pos_out[base + lo + x] = p[i];
  }
}

struct MoveArgs {
  uint8_t *k, *v;
  int64_t seq, row, head;  // bytes
  int chunks;              // 16-byte chunks of a row of one head
  int blocks;              // workgroups of a (sequence, head); 0: the short form moves by itself
};

// The n moves of a head by threads i0 < step: 16-byte chunks of K and V, kMoves at
// a time, non-temporal (15,360 rows of eight heads: 26.5 us against 32.5).
__device__ __forceinline__ void move_rows(const EvictArgs& a, const MoveArgs& t, const RowInfo& r, int bh,
                                          int n, int64_t i0, int64_t step) {
  constexpr int kMoves = 4;
  const int64_t base = (int64_t)bh * a.C;
  const int64_t off = r.b * t.seq + (bh % a.Hkv) * t.head;
  const int64_t total = (int64_t)n * t.chunks;
  for (; i0 < total; i0 += kMoves * step) {
    int64_t d[kMoves];
    u32x4 kx[kMoves], vx[kMoves];
#pragma unroll
    for (int e = 0; e < kMoves; ++e) {
      const int64_t i = min(i0 + e * step, total - 1);  // past the end: the last again, not stored
      const int mv = (int)(i / t.chunks), ch = (int)(i - (int64_t)mv * t.chunks);
      const int dst = a.holes[(int64_t)bh * a.half + mv], src = a.movers[(int64_t)bh * a.half + mv];
      const int64_t s = off + src * t.row + 16 * ch;
      d[e] = off + dst * t.row + 16 * ch;
      kx[e] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(t.k + s));
      vx[e] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(t.v + s));
      if (ch == 0 && i0 + e * step < total) {
        a.w_out[base + dst] = a.w[base + src];
        a.pos_out[base + dst] = position(a, r, base, src);
      }
    }
#pragma unroll
    for (int e = 0; e < kMoves; ++e) {
      if (i0 + e * step >= total) continue;
      __builtin_nontemporal_store(kx[e], reinterpret_cast<u32x4*>(t.k + d[e]));
      __builtin_nontemporal_store(vx[e], reinterpret_cast<u32x4*>(t.v + d[e]));
    }
  }
}

constexpr int kMoveThreads = 256;
// The heads of a row lie next to each other in most caches, and so do their
// workgroups here.
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a, MoveArgs t) {
  const int heads = a.B * a.Hkv;
  const int bh = blockIdx.x % heads, x = blockIdx.x / heads;
  const int n = a.moves[bh];
  if (n == 0) return;
  const RowInfo r = row_info(a, bh);
  move_rows(a, t, r, bh, n, (int64_t)x * kMoveThreads + threadIdx.x, (int64_t)t.blocks * kMoveThreads);
}

// A whole head, P rows a thread; with t.blocks = 0 its moves too.
template <int P, int NT>
__global__ __launch_bounds__(NT) void evict_short_kernel(EvictArgs a, MoveArgs t) {
  __shared__ uint32_t h[kDigits][kBins], keep_s[NT];
  __shared__ int part[NT / 64], pick[2];
  const int bh = blockIdx.x;
  const RowInfo r = row_info(a, bh);
  const int64_t base = (int64_t)bh * a.C;
  if (bh % a.Hkv == 0 && threadIdx.x == 0) a.lens_out[r.b] = min(r.L, a.budget);
  Rows<P> x;
  const int first = threadIdx.x * P;
  load_rows<P>(a, r, base, first, r.L, x);
  uint32_t keep = ~0u;
  if (r.L > a.budget) {
    for (int i = threadIdx.x; i < kDigits * kBins; i += NT) (&h[0][0])[i] = 0;
    __syncthreads();
    Cut cut{0u, a.budget};
#pragma unroll
    for (int pass = 0; pass < kDigits; ++pass) {
      count_digits<P>(x, cut.prefix, pass, h[pass]);
      __syncthreads();
      int cnt[kBins / NT];
#pragma unroll
      for (int i = 0; i < kBins / NT; ++i) cnt[i] = (int)h[pass][kBins - 1 - (threadIdx.x * (kBins / NT) + i)];
      cut = narrow<NT>(cut, cnt, pass, part, pick);
    }
    const int left = cut.need - block_scan<NT>(equal_rows<P>(x, cut.prefix), part).before;
    keep = staying<P>(x, cut.prefix, left);
  }
  // Holes below the budget in the low half, movers from it on in the high half:
  // at most kShortRows / 2 of each.
  int both = 0;
#pragma unroll
  for (int i = 0; i < P; ++i)
    if (i < x.n && (first + i < a.budget) != (keep >> i & 1)) both += first + i < a.budget ? 1 : 1 << 16;
  const Scan s = block_scan<NT>(both, part);
  if (threadIdx.x == 0) a.moves[bh] = s.all & 0xffff;
  int at = s.before & 0xffff, am = s.before >> 16;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (i >= x.n) continue;
    const int j = first + i;
    const bool stay = keep >> i & 1;
    if (j < a.budget && !stay) a.holes[(int64_t)bh * a.half + at++] = j;
    if (j >= a.budget && stay) a.movers[(int64_t)bh * a.half + am++] = j;
  }
  keep_s[threadIdx.x] = keep;
  __syncthreads();
  const int hi = min(r.L, a.budget);
  if (hi > 0) write_kept<P, NT>(a, r, base, 0, hi, keep_s);
  // (The lists were written by this workgroup, ahead of the barrier.)
  if (t.blocks == 0) move_rows(a, t, r, bh, s.all & 0xffff, threadIdx.x, NT);
}

// The bins of a thread in histogram `pass` of a chunk, from the top.
__device__ __forceinline__ u16x4 chunk_bins(const EvictArgs& a, int bh, int pass, int chunk) {
  static_assert(kBins / kThreads == 4 && digit_mask(kDigits - 1) == 16 * 64 - 1, "bins of a thread, of a lane");
  const int64_t at = (((int64_t)pass * a.B * a.Hkv + bh) * a.chunks + chunk) * kBins;
  const u16x4 v = *reinterpret_cast<const u16x4*>(a.hist + at + kBins - 4 - 4 * threadIdx.x);
  return u16x4{v[3], v[2], v[1], v[0]};
}

// The cut after `passes` passes: the last histogram, added up over the chunks,
// narrows the cut stored by the launch before; the first workgroup of a head
// stores the new one.
__device__ __forceinline__ Cut cut_after(const EvictArgs& a, int bh, int passes, int* part, int* pick) {
  Cut cut{0u, a.budget};
  if (passes == 0) return cut;
  int cnt[4] = {0, 0, 0, 0};
#pragma unroll 16
  for (int x = 0; x < a.chunks; ++x) {
    const u16x4 v = chunk_bins(a, bh, passes - 1, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) cnt[i] += v[i];
  }
  if (passes > 1) cut = a.cuts[bh * kDigits + passes - 2];
  cut = narrow<kThreads>(cut, cnt, passes - 1, part, pick);
  if (blockIdx.x % a.chunks == 0 && threadIdx.x == 0) a.cuts[bh * kDigits + passes - 1] = cut;
  return cut;
}

// Histogram of digit PASS of a chunk's keys that share the digits before it.
template <int PASS>
__global__ __launch_bounds__(kThreads) void evict_hist_kernel(EvictArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t h[kBins];
  __shared__ int part[kThreads / 64], pick[2];
  const int bh = blockIdx.x / a.chunks, x = blockIdx.x - bh * a.chunks;
  const RowInfo r = row_info(a, bh);
  if (r.L <= a.budget) return;
  const Chunk c = chunk_of(a, x, r.L);
  const int64_t base = (int64_t)bh * a.C;
  Rows<kPer> rows;
  load_rows<kPer>(a, r, base, c.lo + threadIdx.x * kPer, c.hi, rows);
  for (int i = threadIdx.x; i < kBins; i += kThreads) h[i] = 0;
  const Cut cut = cut_after(a, bh, PASS, part, pick);
  __syncthreads();
  int over = 0;  // rows above the prefix
  for (int lo = c.lo;;) {
    count_digits<kPer>(rows, cut.prefix, PASS, h);
    if constexpr (PASS == kDigits - 1)
#pragma unroll
      for (int i = 0; i < kPer; ++i) over += i < rows.n && (rows.key[i] & prefix_mask(PASS)) > cut.prefix;
    lo += kPart;
    if (lo >= c.hi) break;
    load_rows<kPer>(a, r, base, lo + threadIdx.x * kPer, c.hi, rows);
  }
  if constexpr (PASS == kDigits - 1) {
    const int all = block_scan<kThreads>(over, part).all;
    if (threadIdx.x == 0) a.above[(int64_t)bh * a.chunks + x] = all;
  }
  __syncthreads();
  const int64_t at = (((int64_t)PASS * a.B * a.Hkv + bh) * a.chunks + x) * kBins;
  const u32x4 v = *reinterpret_cast<const u32x4*>(h + 4 * threadIdx.x);
  *reinterpret_cast<u16x4*>(a.hist + at + 4 * threadIdx.x) =
      u16x4{(uint16_t)v[0], (uint16_t)v[1], (uint16_t)v[2], (uint16_t)v[3]};
}

// Which rows of a chunk stay, and the holes or movers among them.
__global__ __launch_bounds__(kThreads) void evict_plan_kernel(EvictArgs a) {
  __shared__ int part[kThreads / 64], pick[2];
  __shared__ int over_s[kThreads], eq_s[kThreads], mine[2];
  __shared__ uint32_t keep_s[kThreads];
  __shared__ uint16_t list_s[kPart];
  const int bh = blockIdx.x / a.chunks, x = blockIdx.x - bh * a.chunks;
  const RowInfo r = row_info(a, bh);
  const Chunk c = chunk_of(a, x, r.L);
  const int64_t base = (int64_t)bh * a.C;
  const bool lower = x < a.chunks_a;
  if (x == 0 && bh % a.Hkv == 0 && threadIdx.x == 0) a.lens_out[r.b] = min(r.L, a.budget);
  if (r.L <= a.budget) {
    for (int j = c.lo + threadIdx.x; j < c.hi; j += kThreads) {
      a.w_out[base + j] = a.w[base + j];
      a.pos_out[base + j] = position(a, r, base, j);
    }
    if (x == 0 && threadIdx.x == 0) a.moves[bh] = 0;
    return;
  }
  Rows<kPer> rows;
  load_rows<kPer>(a, r, base, c.lo + threadIdx.x * kPer, c.hi, rows);
  const Cut cut = cut_after(a, bh, kDigits, part, pick);
  const int bin = (int)(cut.prefix & digit_mask(kDigits - 1));
  // Over the chunks before this one: rows with the cut's key and, with how many
  // of those stay in each, the holes or movers.
  int eq_before = 0, before = 0, all = 0, eq_run = 0;
  for (int i0 = 0; i0 < a.chunks; i0 += kThreads) {
    const int cn = min(kThreads, a.chunks - i0), i = i0 + threadIdx.x;
    __syncthreads();
    over_s[threadIdx.x] = i < a.chunks ? a.above[(int64_t)bh * a.chunks + i] : 0;
    eq_s[threadIdx.x] = 0;
    __syncthreads();
    // A wave takes a chunk's histogram (the last digit has 1,024 bins), 16 bins a
    // lane; the chunks of a wave are read together, kEach at a time.  Few rows
    // share all the digits before, so most lanes find nothing.
    constexpr int kEach = 5;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int y0 = wave; y0 < cn; y0 += kEach * (kThreads / 64)) {
      u32x4 v[kEach][2];
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int y = min(y0 + e * (kThreads / 64), cn - 1);
        const int64_t at = (((int64_t)(kDigits - 1) * a.B * a.Hkv + bh) * a.chunks + i0 + y) * kBins;
        v[e][0] = *reinterpret_cast<const u32x4*>(a.hist + at + 16 * lane);
        v[e][1] = *reinterpret_cast<const u32x4*>(a.hist + at + 16 * lane + 8);
      }
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int y = y0 + e * (kThreads / 64);
        const u32x4 any = v[e][0] | v[e][1];
        if (y >= cn || (any[0] | any[1] | any[2] | any[3]) == 0 || 16 * lane + 15 < bin) continue;
        int over = 0, eq = 0;
#pragma unroll
        for (int i2 = 0; i2 < 16; ++i2) {
          const int n = (int)(v[e][i2 >> 3][(i2 >> 1) & 3] >> 16 * (i2 & 1) & 0xffffu);
          over += 16 * lane + i2 > bin ? n : 0;
          eq += 16 * lane + i2 == bin ? n : 0;
        }
        if (over != 0) atomicAdd(&over_s[y], over);
        if (eq != 0) eq_s[y] = eq;  // one lane has the bin
      }
    }
    __syncthreads();
    const int over = over_s[threadIdx.x], eq = eq_s[threadIdx.x];
    const Scan e = block_scan<kThreads>(eq, part);
    const int stay = over + min(max(cut.need - eq_run - e.before, 0), eq);
    int cnt = 0;
    if (i < a.chunks && (i < a.chunks_a) == lower) {
      const Chunk ci = chunk_of(a, i, r.L);
      cnt = lower ? ci.hi - ci.lo - stay : stay;
    }
    const Scan s = block_scan<kThreads>(cnt, part);
    if (i == x) {
      mine[0] = eq_run + e.before;
      mine[1] = all + s.before;
    }
    eq_run += e.all;
    all += s.all;
  }
  __syncthreads();
  eq_before = mine[0];
  before = mine[1];
  if (x == 0 && threadIdx.x == 0) a.moves[bh] = all;  // holes
  int32_t* list = (lower ? a.holes : a.movers) + (int64_t)bh * a.half;
  for (int lo = c.lo;;) {
    const Scan e = block_scan<kThreads>(equal_rows<kPer>(rows, cut.prefix), part);
    const uint32_t keep = staying<kPer>(rows, cut.prefix, cut.need - eq_before - e.before);
    int listed = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) listed += i < rows.n && lower != (keep >> i & 1);
    const Scan s = block_scan<kThreads>(listed, part);
    __syncthreads();  // the last part's list and bits may still be in use
    int at = s.before;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < rows.n && (bool)(keep >> i & 1) != lower) list_s[at++] = (uint16_t)(threadIdx.x * kPer + i);
    keep_s[threadIdx.x] = keep;
    __syncthreads();
    for (int i = threadIdx.x; i < s.all; i += kThreads) list[before + i] = lo + list_s[i];
    if (lower && lo < c.hi) write_kept<kPer, kThreads>(a, r, base, lo, c.hi, keep_s);
    eq_before += e.all;
    before += s.all;
    lo += kPart;
    if (lo >= c.hi) break;
    load_rows<kPer>(a, r, base, lo + threadIdx.x * kPer, c.hi, rows);
  }
}

// Bound by its launch and a few dependent loads: 5.2 us for 24 layers of eight heads
// of 128, at most 64 rows a path (2 MB).
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
    u32x4 x[8];
    int src[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int p = j0 + e < a.P ? path[j0 + e] : -1;
      on = on && p > last && p < room;
      src[e] = on ? p : -1;
      if (on) {
        last = p;
        ++n;
        if (moves && p != j0 + e) x[e] = *reinterpret_cast<const u32x4*>(base + p * a.row);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (moves && src[e] >= 0 && src[e] != j0 + e)
        *reinterpret_cast<u32x4*>(base + (j0 + e) * a.row) = x[e];
  }
  if (a.lens_out && hc == 0 && blockIdx.y == 0 && blockIdx.z == 0)
    a.lens_out[b] = past < 0 ? past : past + n;
}

struct Layout {
  int chunk, chunks_max, half;
  size_t hist, cuts, above, list, moves, total;
};
Layout layout_of(int B, int Hkv, int C) {
  Layout y{};
  const size_t bh = (size_t)B * Hkv;
  // Chunks of the long form: some 32 a head, each WG adds up all of them.
  const int64_t parts = std::min<int64_t>(kParts, (C + 32LL * kPart - 1) / (32LL * kPart));
  y.chunk = (int)(parts * kPart);
  y.chunks_max = (int)(((int64_t)C + y.chunk - 1) / y.chunk + 1);  // whatever the budget
  y.half = C / 2 + 1;  // moves: at most min(budget, C - budget)
  auto up = [](size_t n) { return (n + 15) / 16 * 16; };
  if (C > kShortRows) {
    y.hist = up(kDigits * bh * y.chunks_max * kBins * sizeof(uint16_t));
    y.cuts = up(bh * kDigits * sizeof(Cut));
    y.above = up(bh * y.chunks_max * 4);
  }
  y.list = up(bh * y.half * 4);
  y.moves = up(bh * 4);
  y.total = y.hist + y.cuts + y.above + 2 * y.list + y.moves;
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
  a.chunk = y.chunk;
  a.chunks_a = (int)(((int64_t)p.budget + y.chunk - 1) / y.chunk);
  a.chunks = a.chunks_a + (int)(((int64_t)p.C - p.budget + y.chunk - 1) / y.chunk);
  a.lens = p.lens;
  a.kept = p.kept;
  a.ends = p.ends;
  a.w = p.w;
  a.pos = p.pos;
  a.w_out = p.w_out;
  a.pos_out = p.pos_out;
  a.lens_out = p.lens_out;
  uint8_t* at = static_cast<uint8_t*>(ws);
  a.hist = reinterpret_cast<uint16_t*>(at);
  a.cuts = reinterpret_cast<Cut*>(at += y.hist);
  a.above = reinterpret_cast<int32_t*>(at += y.cuts);
  a.holes = reinterpret_cast<int32_t*>(at += y.above);
  a.movers = reinterpret_cast<int32_t*>(at += y.list);
  a.moves = reinterpret_cast<int32_t*>(at += y.list);
  a.half = y.half;
  MoveArgs t;
  t.k = static_cast<uint8_t*>(p.k);
  t.v = static_cast<uint8_t*>(p.v);
  t.seq = p.seq * p.elem;
  t.row = p.row * p.elem;
  t.head = p.head * p.elem;
  t.chunks = p.D * p.elem / 16;
  const int64_t most = (int64_t)std::min(p.budget, p.C - p.budget) * t.chunks;  // of a head
  t.blocks = (int)std::max<int64_t>(1, std::min<int64_t>((most + kMoveThreads - 1) / kMoveThreads, std::max(1, 2048 / bh)));
  if (p.C <= kShortRows) {
    if (most <= kFewMoves) t.blocks = 0;
    auto whole = [&](auto kernel, int threads) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)bh), dim3(threads), 0, s, a, t);
    };
    if (p.C <= 4096) whole(evict_short_kernel<8, 512>, 512);
    else if (p.C <= 8192) whole(evict_short_kernel<8, 1024>, 1024);
    else whole(evict_short_kernel<16, 1024>, 1024);
  } else {
    const dim3 grid((unsigned)(bh * a.chunks)), block(kThreads);
    if (p.C > p.budget) {
      hipLaunchKernelGGL(evict_hist_kernel<0>, grid, block, 0, s, a);
      hipLaunchKernelGGL(evict_hist_kernel<1>, grid, block, 0, s, a);
      hipLaunchKernelGGL(evict_hist_kernel<2>, grid, block, 0, s, a);
    }
    hipLaunchKernelGGL(evict_plan_kernel, grid, block, 0, s, a);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.C <= p.budget || t.blocks == 0) return e;
  hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)(bh * t.blocks)), dim3(kMoveThreads), 0, s, a, t);
  return hipGetLastError();
}

hipError_t launch_cache_commit(const CommitArgs& a, int layers, hipStream_t s) {
  const int64_t threads = (int64_t)a.B * a.Hkv * a.chunks;
  const dim3 grid((unsigned)((threads + 255) / 256), (unsigned)std::max(1, layers), layers > 0 ? 2 : 1);
  hipLaunchKernelGGL(cache_commit_kernel, grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace lc
