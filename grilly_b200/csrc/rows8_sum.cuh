// Joins the column sums that blocks of rows left in a workspace.
#pragma once
#include <cuda_runtime.h>

namespace gb {

// out[f] = sum over the blocks of partial[block][f], always in the same order, for 32 columns: 512 threads, 16 per column
// over every 16th block, added up in turn.
__device__ __forceinline__ void column_total(const float* partial, float* out, int blocks, int F, int which, float (&part)[16][33]) {
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int f = which * 32 + tx;
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
