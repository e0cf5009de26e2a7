// Joins the column sums that blocks of rows left in a workspace; launches of a kernel that follows another of the same call.
#pragma once
#include <cuda_runtime.h>

namespace gb {

// A kernel that follows another one of the same call is launched and set up while that one ends (2 us a launch), and waits
// here before it reads what the other wrote (with ordinary loads: it changed during this kernel's life).
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
inline cudaLaunchAttribute early_launch() {
  cudaLaunchAttribute a = {};
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  return a;
}
template <class... P, class... A>
cudaError_t launch_following(cudaStream_t stream, void (*kern)(P...), unsigned grid, unsigned block, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr = early_launch();
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(block, 1, 1);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// out[f] = sum over the blocks of partial[block][f], always in the same order, for 32 columns: 512 threads, 16 per column
// over every 16th block, added up in turn.
__device__ __forceinline__ void column_total(const float* partial, float* out, int blocks, int F, int which, float (&part)[16][33]) {
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int f = which * 32 + tx;
  float acc = 0.f;
  if (f < F) {
#pragma unroll 4
    for (int b = ty; b < blocks; b += 16) acc += partial[static_cast<long long>(b) * F + f];
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
