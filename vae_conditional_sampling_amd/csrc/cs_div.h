// n / d for any 32-bit n by a multiplication (the round-up form of Granlund and Montgomery, 1994), d from 1 to 2^32 - 1: a
// 64-bit division by a size of the call costs a lane several hundred instructions, a 32-bit one about forty.  Also grids of more
// workgroups than a launch's first axis may hold, and rows in memory that must not meet.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

struct CsDiv {
  uint32_t d, mul, s1, s2;
};
inline CsDiv cs_div_by(int64_t d) {
  uint32_t l = 0;
  while (l < 32 && (1ull << l) < (uint64_t)d) ++l;
  const uint64_t mul = ((1ull << 32) * ((1ull << l) - (uint64_t)d)) / (uint64_t)d + 1;
  return CsDiv{(uint32_t)d, (uint32_t)mul, l ? 1u : 0u, l ? l - 1 : 0u};
}
__device__ __forceinline__ uint32_t cs_div(uint32_t n, const CsDiv& d) {   // (scalar instructions where n is uniform)
  const uint32_t t = __umulhi(n, d.mul);
  return (t + ((n - t) >> d.s1)) >> d.s2;
}

// Workgroups of up to 1024 threads in two axes (an axis of a launch has to stay below 2^32 threads), and the number of one;
// the last row may hold up to 2^20 - 1 more workgroups than were asked for.  The number has 32 bits: callers stay at 2^31.
constexpr int CS_GRID_SHIFT = 20;
inline dim3 cs_grid(int64_t blocks) {
  constexpr int64_t ROW = 1ll << CS_GRID_SHIFT;
  return blocks <= ROW ? dim3((unsigned)blocks) : dim3((unsigned)ROW, (unsigned)((blocks + ROW - 1) >> CS_GRID_SHIFT));
}
__device__ __forceinline__ uint32_t cs_block() { return (blockIdx.y << CS_GRID_SHIFT) + blockIdx.x; }

// Rows of `row` units along three axes: the units from the first one's start to the last one's end, or -1 where rows may meet (from
// the closest axis on, every stride has to clear what lies within).
inline int64_t cs_rows_apart(const int64_t n[3], const int64_t stride[3], int64_t row) {
  int order[3] = {0, 1, 2};
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j)
      if (stride[order[j]] > stride[order[j + 1]]) { const int t = order[j]; order[j] = order[j + 1]; order[j + 1] = t; }
  int64_t end = row;
  for (int i = 0; i < 3; ++i) {
    const int a = order[i];
    if (n[a] <= 1) continue;
    if (stride[a] < end) return -1;
    end += (n[a] - 1) * stride[a];
  }
  return end;
}
