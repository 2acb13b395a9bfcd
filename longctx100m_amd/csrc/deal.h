// How the keys of a ragged batch are dealt over the workgroups, on the device:
// the host fixes the number of slots (and with it a workspace), the lengths are
// read here.  A slot holds `per` tiles of one sequence, the fewest with which the
// slots suffice for all, so a batch of unequal lengths loads the chip evenly.
//
// rows(b) is the number of keys of sequence b, below 2^30; TILE keys are a tile.
#pragma once

#include "cache.h"
#include "common.h"

namespace lc {

constexpr int kTile = 64;  // keys by which a sequence is dealt out

// Tiles of a sequence, at least one (so that every sequence has a slot).
template <int TILE>
__device__ __forceinline__ int tiles_of(int rows) {
  return max(1, (rows + TILE - 1) / TILE);
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
// even shares, and ceil(tiles / per) adds less than one each.  As many slots as
// sequences: a slot is a whole sequence.
template <int TILE, typename Rows>
__device__ __forceinline__ int slot_tiles(const Rows& rows, int B, int slots) {
  const int lane = threadIdx.x & 63;
  if (B == 1) return (tiles_of<TILE>(rows(0)) + slots - 1) / slots;
  if (slots == B) return (1 << 30) / TILE;
  if (B > kTightBatch) {
    int total = 0;
    for (int b0 = 0; b0 < B; b0 += 64)
      total += wave_sum_i(b0 + lane < B ? tiles_of<TILE>(rows(b0 + lane)) : 0);
    return (total + slots - B - 1) / (slots - B);
  }
  const int mine = lane < B ? tiles_of<TILE>(rows(lane)) : 0;
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
// every sequence's first slot and its slots in deal [B].
template <int TILE = kTile, typename Rows>
__device__ __forceinline__ bool share_of(const Rows& rows, int B, int slots, int2* deal, int slot,
                                         Share& s) {
  const int lane = threadIdx.x & 63;
  const int per = slot_tiles<TILE>(rows, B, slots);
  const float inv = 1.f / (float)per;
  int first = 0, at = -1;  // of sequence at
  int base = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    const int b = b0 + lane;
    const int n = b < B ? slots_for(tiles_of<TILE>(rows(b)), per, inv) : 0;
    const int end = base + wave_scan(n);
    if (blockIdx.x == 0 && threadIdx.x < 64 && b < B) deal[b] = make_int2(end - n, n);
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
  const int n = rows(s.b);
  s.k0 = __builtin_amdgcn_readfirstlane(min((slot - first) * per * TILE, n));
  s.k1 = __builtin_amdgcn_readfirstlane(min(n - s.k0, per * TILE)) + s.k0;
  return true;
}

// The same with slots that do not end where a sequence does: the tiles of all
// sequences one behind another, every slot the same number of them, `least` at
// least.  A slot's run of one sequence's tiles is a segment, number slot + b (each
// step of either starts one, so slots + B numbers suffice).
//   for (Spans<TILE, Rows> s(...); s.next();) ... s.b, s.k0, s.k1, s.segment
// visits a slot's segments, the whole workgroup together; a sequence without keys
// has none.  The first workgroup leaves every sequence's first segment and its
// segments in deal [B].  whole: slot b is sequence b, also one without keys.
template <int TILE, typename Rows>
struct Spans {
  const Rows& rows;
  int B, slot;
  bool whole;
  int2* deal;
  int per, t0, t1;
  int b0, base, mine, end;  // of the 64 sequences from b0 on, over the lanes
  uint64_t left;            // those still to visit
  int b, k0, k1, segment;

  __device__ __forceinline__ static int tiles(int n) { return (n + TILE - 1) / TILE; }
  __device__ __forceinline__ Spans(const Rows& rows_, int B_, int slots, bool whole_, int least, int2* deal_,
                                   int slot_)
      : rows(rows_), B(B_), slot(slot_), whole(whole_), deal(deal_) {
    const int lane = threadIdx.x & 63;
    b0 = -64;
    base = 0;
    left = 0;
    per = t0 = t1 = 0;
    if (whole) return;
    int all = 0;
    if (B == 1) all = tiles(rows(0));
    else
      for (int x = 0; x < B; x += 64) all += wave_sum_i(x + lane < B ? tiles(rows(x + lane)) : 0);
    per = __builtin_amdgcn_readfirstlane(max((all + slots - 1) / slots, least));
    t0 = slot * per;
    t1 = min(t0 + per, all);
  }
  __device__ __forceinline__ bool next() {
    if (whole) {
      if (b0 >= 0) return false;
      b0 = 0;
      b = slot;
      k0 = 0;
      k1 = __builtin_amdgcn_readfirstlane(rows(b));
      segment = b;
      return true;
    }
    const int lane = threadIdx.x & 63;
    while (left == 0) {
      b0 += 64;
      if (b0 >= B || (base >= t1 && blockIdx.x != 0)) return false;
      mine = b0 + lane < B ? tiles(rows(b0 + lane)) : 0;
      end = base + wave_scan(mine);
      if (blockIdx.x == 0 && threadIdx.x < 64 && b0 + lane < B) {
        const int first = (end - mine) / per, last = mine > 0 ? (end - 1) / per : first - 1;
        deal[b0 + lane] = make_int2(first + b0 + lane, last - first + 1);
      }
      left = __ballot(mine > 0 && end > t0 && end - mine < t1);
      base = __builtin_amdgcn_readlane(end, 63);
    }
    const int x = __ffsll((unsigned long long)left) - 1;
    left &= left - 1;
    b = b0 + x;
    segment = slot + b;
    const int stop = __builtin_amdgcn_readlane(end, x), start = stop - __builtin_amdgcn_readlane(mine, x);
    const int n = __builtin_amdgcn_readfirstlane(rows(b));
    k0 = max(t0 - start, 0) * TILE;
    k1 = stop <= t1 ? n : (t1 - start) * TILE;
    return true;
  }
};

}  // namespace lc
