// Sum of a few hundred partial rows, column by column and in a fixed order: the second half of the reductions over tokens.
#pragma once

#include "common.cuh"

namespace tmoe {

constexpr int kColumnSumThreads = 1024;   // 32 columns x 32 rows of threads

// The sum of partial[b, col], b < rows, for this thread's column, valid in the first warp; every block thread calls it.  32 rows of threads
// keep 148 partial rows to five loads in flight a thread (with eight rows of threads the loop alone took 5 us).
__device__ __forceinline__ float column_sum(const float *__restrict__ partial, int rows, int n, int col, float (&part)[32][33]) {
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  float s = 0.f;
  if (col < n) {
#pragma unroll 8
    for (int b = row; b < rows; b += 32) s += partial[(int64_t)b * n + col];
  }
  part[row][lane] = s;
  __syncthreads();
  float t = 0.f;
  if (row == 0) {
#pragma unroll
    for (int i = 0; i < 32; ++i) t += part[i][lane];
  }
  return t;
}

}  // namespace tmoe
