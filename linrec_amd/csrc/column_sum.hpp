// Sums over the rows of a dense fp32 matrix, in an order that depends on its sizes alone: how gradients of parameters that all
// positions share are put together from the workgroups' partial sums.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "layer_common.hpp"

namespace linrec {

constexpr int SUM_WAVES = 16;
constexpr int64_t SUM_ROWS = 512;  // rows a workgroup sums before a second launch pays

inline int64_t column_sum_chunks(int64_t rows) { return rows <= 2 * SUM_ROWS ? 1 : cdiv(rows, SUM_ROWS); }

// A workgroup sums `per_chunk` rows of 64 columns; finish(column, sum) where it has them all, else row blockIdx.y of `out`.
template <typename F>
__device__ __forceinline__ void column_sum_block(const float* in, int64_t rows, int64_t columns, int64_t per_chunk, F&& finish) {
  __shared__ float sh[SUM_WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = int64_t(blockIdx.x) * 64 + lane;
  const int64_t first = int64_t(blockIdx.y) * per_chunk, end = first + per_chunk < rows ? first + per_chunk : rows;
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < columns) {
    int64_t r = first + wave;
    for (; r + 3 * SUM_WAVES < end; r += 4 * SUM_WAVES) {
#pragma unroll
      for (int q = 0; q < 4; ++q) s[q] += in[(r + q * SUM_WAVES) * columns + c];
    }
    for (; r < end; r += SUM_WAVES) s[0] += in[r * columns + c];
  }
  sh[wave][lane] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (wave == 0 && c < columns) {
    float t = sh[0][lane];
#pragma unroll
    for (int w = 1; w < SUM_WAVES; ++w) t += sh[w][lane];
    finish(c, t);
  }
}

}  // namespace linrec
