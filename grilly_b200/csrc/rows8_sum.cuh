// Joins the column sums that blocks of rows left in a workspace.
#pragma once
#include <cuda_runtime.h>

namespace gb {

// out[f] = sum over the blocks of partial[block][f], always in the same order: 32 columns per block of 512 threads, 16
// threads per column over every 16th block, added up in turn.
static __global__ void __launch_bounds__(512) sum_partials_kernel(const float* __restrict__ partial, float* __restrict__ out, int blocks, int F) {
  __shared__ float part[16][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int f = blockIdx.x * 32 + tx;
  float acc = 0.f;
  if (f < F) {
#pragma unroll 4
    for (int b = ty; b < blocks; b += 16) acc += __ldg(partial + static_cast<long long>(b) * F + f);
  }
  part[ty][tx] = acc;
  __syncthreads();
  if (ty == 0 && f < F) {
#pragma unroll
    for (int i = 1; i < 16; ++i) acc += part[i][tx];
    out[f] = acc;
  }
}

}  // namespace gb
