// Rotary positions of [batch, tokens, heads, head_dim] rows (gfx950), forward and
// backward: out = factor R(position) x, or factor R(position)^T x.
//
// Bound by the bytes of x and out: 32,768 tokens of 40 heads of 128 in bf16 move 671 MB
// in 128 us (5.2 TB/s, a copy's rate), a million of 8 heads of 128 4.3 GB in 740 (5.8).  The
// (cos, sin) of a token's pairs are formed once, in LDS, and serve all its heads; a
// thread turns N pairs at a time, eight where 16 bytes a load fit, the next ones on
// their way.  Four tokens of few heads are less than a workgroup's threads could take, and
// latency bounds it: 2 and 3 heads of 128 run at 2.9 and 3.3 TB/s, of 64 at 1.5 and 2.2, 8
// of 64 at 4.6.
#include "rotary.h"

#include <type_traits>

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

template <typename T, int N>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  __shared__ float2 cs[kTurnTokens * kTurnPairs];
  const uint32_t row0 = blockIdx.x * (uint32_t)a.group;
  const int n = (int)min((uint32_t)a.group, a.rows - row0);
  auto at = [&](const HeadRows& s, int t) {
    const uint32_t row = row0 + t, b = row / a.tokens;
    return (int64_t)b * s.seq + (int64_t)(row - b * a.tokens) * s.token;
  };
  turn_tokens<T, N, (N > 1)>(
      cs, a.turns, n, a.heads, a.D, a.xs.head, a.os.head, a.copy, a.sign,
      [&](int t) { return static_cast<const T*>(a.x) + at(a.xs, t); },
      [&](int t) { return static_cast<T*>(a.out) + at(a.os, t); },
      [&](int t) { return a.positions ? a.positions[row0 + t] : a.pos0 + (row0 + t) % a.tokens; },
      [](int) { return true; });
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
  const unsigned grid = (a.rows + a.group - 1) / a.group;
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, s, a); };
  auto by_type = [&](auto n) {
    constexpr int N = decltype(n)::value;
    if (p.dtype == 1) launch(rotary_kernel<uint16_t, N>);
    else launch(rotary_kernel<float, N>);
  };
  // The widest accesses that pairs, heads and addresses allow: eight pairs a thread, four
  // (32,768 tokens of 40 heads of 80 dims, 40 of which turn: 91 us, 4.6 TB/s; one pair
  // at a time, its angle formed for each head, took 326) or one (heads of 128, 100 of
  // which turn: 217 us, 3.1 TB/s, 2-byte accesses; 449).
  const int half = p.turns.half;
  if (half % 8 == 0 && p.D % 16 == 0 && p.align >= 16) by_type(std::integral_constant<int, 8>{});
  else if (half % 4 == 0 && p.D % 8 == 0 && p.align >= (p.dtype == 1 ? 8 : 16)) by_type(std::integral_constant<int, 4>{});
  else by_type(std::integral_constant<int, 1>{});
  return hipGetLastError();
}

}  // namespace lc
