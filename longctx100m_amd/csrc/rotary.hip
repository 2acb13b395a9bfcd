// Rotary positions of [batch, tokens, heads, head_dim] rows (gfx950), forward and
// backward: out = factor R(position) x, or factor R(position)^T x.
//
// Bound by the bytes of x and out: 32,768 tokens of 40 heads of 128 in bf16 move 671 MB
// in 128 us (5.2 TB/s, a copy's rate).  The (cos, sin) of a token's pairs are formed
// once, in LDS, and serve all its heads; a thread turns eight pairs at a time,
// 16 bytes a load, the next ones on their way.
#include "rotary.h"

#include <algorithm>

namespace lc {
namespace {

struct RotaryArgs {
  Turns turns;
  uint32_t rows, tokens;  // rows = batch * tokens, below 2^24
  int group, heads, D;
  bool copy;
  uint64_t sign;
  const int64_t* positions;
  int64_t pos0;
  const void* x;
  void* out;
  HeadRows xs, os;
};

template <typename T, bool kVec>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  __shared__ float2 cs[kTurnTokens * kTurnPairs];
  const uint32_t row0 = blockIdx.x * (uint32_t)a.group;
  const int n = (int)min((uint32_t)a.group, a.rows - row0);
  auto at = [&](const HeadRows& s, int t) {
    const uint32_t row = row0 + t, b = row / a.tokens;
    return (int64_t)b * s.seq + (int64_t)(row - b * a.tokens) * s.token;
  };
  turn_tokens<T, kVec>(
      cs, a.turns, n, a.heads, a.D, a.xs.head, a.os.head, a.copy, a.sign,
      [&](int t) { return static_cast<const T*>(a.x) + at(a.xs, t); },
      [&](int t) { return static_cast<T*>(a.out) + at(a.os, t); },
      [&](int t) { return a.positions ? a.positions[row0 + t] : a.pos0 + (row0 + t) % a.tokens; },
      [](int) { return true; });
}

// Any rotary_dim and head_dim: a thread takes one pair, or one dim that is copied.
template <typename T>
__global__ __launch_bounds__(256) void rotary_any_kernel(RotaryArgs a) {
  const int per = a.turns.half + (a.copy ? a.D - 2 * a.turns.half : 0);
  const int64_t total = (int64_t)a.rows * a.heads * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t rh = i / per;
    const int u = (int)(i - rh * per);
    const uint32_t row = (uint32_t)(rh / a.heads), b = row / a.tokens, t = row - b * a.tokens;
    const int h = (int)(rh - (int64_t)row * a.heads);
    const T* x = static_cast<const T*>(a.x) + (int64_t)b * a.xs.seq + (int64_t)t * a.xs.token + h * a.xs.head;
    T* o = static_cast<T*>(a.out) + (int64_t)b * a.os.seq + (int64_t)t * a.os.token + h * a.os.head;
    if (u >= a.turns.half) {
      o[u + a.turns.half] = x[u + a.turns.half];
      continue;
    }
    const int64_t pos = a.positions ? a.positions[row] : a.pos0 + t;
    const float2 cs = turn_cos_sin(a.sign * (uint64_t)pos * a.turns.turns[u], a.turns.factor);
    const int d0 = a.turns.interleaved ? 2 * u : u, d1 = a.turns.interleaved ? 2 * u + 1 : u + a.turns.half;
    const float p = load_f32(x + d0), q = load_f32(x + d1);
    store_from_f32(o + d0, p * cs.x - q * cs.y);
    store_from_f32(o + d1, q * cs.x + p * cs.y);
  }
}

}  // namespace

hipError_t launch_rotary(const RotaryProblem& p, hipStream_t s) {
  RotaryArgs a;
  a.turns = p.turns;
  a.rows = (uint32_t)(p.batch * p.tokens);
  a.tokens = (uint32_t)p.tokens;
  a.heads = p.heads;
  a.D = p.D;
  a.copy = p.copy;
  a.sign = p.inverse ? ~(uint64_t)0 : 1;
  a.positions = p.positions;
  a.pos0 = p.pos0;
  a.x = p.x;
  a.out = p.out;
  a.xs = p.xs;
  a.os = p.os;
  a.group = a.rows <= 1024 ? 1 : kTurnTokens;
  const bool whole = p.turns.half % 8 == 0 && p.turns.half <= kTurnPairs && p.D % 16 == 0 && p.vec;
  if (whole) {
    const unsigned grid = (a.rows + a.group - 1) / a.group;
    if (p.dtype == 1) hipLaunchKernelGGL((rotary_kernel<uint16_t, true>), dim3(grid), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((rotary_kernel<float, true>), dim3(grid), dim3(256), 0, s, a);
  } else {
    const int64_t items = (int64_t)a.rows * a.heads * (p.D - p.turns.half);
    const unsigned grid = (unsigned)std::min<int64_t>((items + 255) / 256, 1 << 16);
    if (p.dtype == 1) hipLaunchKernelGGL(rotary_any_kernel<uint16_t>, dim3(grid), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(rotary_any_kernel<float>, dim3(grid), dim3(256), 0, s, a);
  }
  return hipGetLastError();
}

}  // namespace lc
