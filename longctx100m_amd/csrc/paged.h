// What the operators of the paged 8-bit cache share: the problem after validation
// and the launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rotary.h"

namespace lc {

// A pool of pages of `rows` tokens: K codes [pages, Hkv, rows, D], V codes
// [pages, Hkv, D, rows], and a scale for K and for V [pages, Hkv].
struct Pool {
  int pages, rows, Hkv, D;
  uint8_t *k, *v;
  float *ks, *vs;
};

struct PagedProblem {
  int B, N, Hq;
  int dtype;  // of q, k, v, out: 0 = f32, 1 = bf16
  Pool pool;
  int width;             // entries of a sequence in the page table
  const int32_t* table;  // [B, width]
  const int32_t* past;   // [B]: rows before the new tokens; < 0: no sequence
  const int32_t* counts;  // [B]: new tokens; null: N
};

struct AppendProblem {
  PagedProblem p;
  Turns turns;
  const void *q, *k, *v;
  void* q_out;
  HeadRows qs, ks, vs;
  bool vec;  // every row of q, k, v and q_out is 16-byte aligned
};
hipError_t launch_paged_append(const AppendProblem& p, hipStream_t s);

size_t paged_attn_bytes(const PagedProblem& p);
hipError_t launch_paged_attn(const PagedProblem& p, const void* q, void* out, float* m, float* l,
                             void* ws, hipStream_t s);

// New tokens of a sequence; 0 where there is no sequence.
__device__ __forceinline__ int new_tokens(const int32_t* counts, int N, int b, int past) {
  int n = N;
  if (counts != nullptr) n = max(0, min(counts[b], N));  // (read along with past, not after it)
  return past < 0 ? 0 : n;
}

}  // namespace lc
