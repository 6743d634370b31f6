// Second half of the column sums over rows (gradients of vectors that every row shares): adds partial sums.
#pragma once

#include "elements.hpp"

namespace tcu {

// out[v][c] = sum over parts of partial[part][v][c], in a fixed order: 64 columns per block, the parts dealt to its waves
struct ColumnSumParams {
  const float *partial;
  float *out[3];
  size_t parts;
  unsigned columns, vectors;  // columns of one vector
};
constexpr int kColumnSumWaves = 8;
__global__ __launch_bounds__(64 * kColumnSumWaves) inline void column_sum_kernel(ColumnSumParams p) {
  __shared__ float lds[kColumnSumWaves * 64];
  const size_t width = (size_t)p.columns * p.vectors, at = (size_t)blockIdx.x * 64 + lane_id();
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (at < width) {
    size_t i = wave_in_block();
    for (; i + 3 * kColumnSumWaves < p.parts; i += 4 * kColumnSumWaves) {
#pragma unroll
      for (int u = 0; u < 4; u++) s[u] += p.partial[(i + u * kColumnSumWaves) * width + at];
    }
    for (; i < p.parts; i += kColumnSumWaves) s[0] += p.partial[i * width + at];
  }
  lds[threadIdx.x] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (threadIdx.x < 64 && at < width) {
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < kColumnSumWaves; w++) t += lds[w * 64 + threadIdx.x];
    p.out[at / p.columns][at % p.columns] = t;
  }
}

}  // namespace tcu
