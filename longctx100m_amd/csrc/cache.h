// What the KV-cache operators share: the problem after validation, launchers,
// and how the past is cut into splits on the device.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lc {

struct CacheProblem {
  int B, N, C, Hq, Hkv, D;
  int dtype;     // 0 = f32, 1 = bf16
  bool precise;  // bf16: the fp32-math kernels
  int64_t seq, row, head;  // strides of K and V in elements
  const int32_t* past;
  const int32_t* parents;  // null: a chain
  float sl2;               // D^-1/2 log2(e)
};

constexpr int kCacheMaxTokens = 256;

size_t cache_attn_bytes(const CacheProblem& p);
hipError_t launch_cache_attn(const CacheProblem& p, const void* q, const void* k, const void* v,
                             void* out, float* m, float* l, void* ws, hipStream_t s);
hipError_t launch_cache_weights(const CacheProblem& p, const void* q, const void* k,
                                const float* m, const float* l, const float* w, float* w_out,
                                hipStream_t s);

struct EvictProblem {
  int B, C, Hkv, D, elem;  // elem: bytes of an element of K and V
  int64_t seq, row, head;
  int budget, sinks, recent;
  const int32_t *lens, *kept, *ends;
  void *k, *v;
  const float* w;
  const int32_t* pos;
  float* w_out;
  int32_t *pos_out, *lens_out;
};
size_t cache_evict_bytes(int B, int Hkv, int C);
hipError_t launch_cache_evict(const EvictProblem& p, void* ws, hipStream_t s);

// One launch takes the caches of this many layers (their pointers are kernel arguments).
constexpr int kCommitLayers = 32;
struct CommitArgs {
  uint8_t* k[kCommitLayers];
  uint8_t* v[kCommitLayers];
  int B, P, C, Hkv, chunks;   // chunks: 16-byte chunks of a row of one head
  int64_t seq, row, head;     // strides in bytes
  const int32_t *past, *path;
  int32_t* lens_out;          // null: not this launch
};
hipError_t launch_cache_commit(const CommitArgs& a, int layers, hipStream_t s);

// Inclusive prefix sum over a wave's lanes with DPP: within the rows of 16 lanes
// by shifts of 1, 2, 4 and 8, then the last lane of row 0 (2) into row 1 (3),
// and lane 31 into the upper half.
template <int kCtrl, int kRows>
__device__ __forceinline__ int dpp_add(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, kCtrl, kRows, 0xf, true);
}
__device__ __forceinline__ int wave_scan(int x) {
  x = dpp_add<0x111, 0xf>(x);
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);
  return dpp_add<0x143, 0xc>(x);
}

}  // namespace lc
