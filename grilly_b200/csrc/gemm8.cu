// Matrix products over 8-bit rows: y = act(s_x s_w x_q W_q^T + b), and the backward pass of a linear layer whose saved
// input is in 8-bit rows. The definitions stand with the entry points in include/grilly_b200.h.
#include "rows8.h"
#include <cuda_bf16.h>
#include <algorithm>

namespace gb {
namespace {

__device__ __forceinline__ float act8(float v, int act) {
  switch (act) {
    case GRILLY_ACT_GELU: {
      const float u = v * fmaf(0.7978845608028654f * 0.044715f, v * v, 0.7978845608028654f);
      return v / (1.f + expf(-2.f * u));
    }
    case GRILLY_ACT_SILU: return v / (1.f + expf(-v));
    case GRILLY_ACT_RELU: return v < 0.f ? 0.f : v;
    default: return v;
  }
}

// One warp per output: 32 lanes walk K in 4-byte words.
template <class T>
__global__ void __launch_bounds__(256) linear_q8_kernel(const int8_t* __restrict__ xq, const float* __restrict__ xs, const int8_t* __restrict__ wq,
                                                        const float* __restrict__ ws, const float* __restrict__ bias, T* y, long long M, int N,
                                                        int K, long long ldx, long long ldw, int act) {
  const int lane = threadIdx.x & 31;
  const long long total = M * N, step = static_cast<long long>(gridDim.x) * 8;
  for (long long o = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); o < total; o += step) {
    const long long m = o / N, n = o % N;
    int acc = 0;
    for (int k = lane; k < K; k += 32) acc += static_cast<int>(xq[m * ldx + k]) * wq[n * ldw + k];
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, s);
    if (lane == 0) {
      float v = static_cast<float>(acc) * xs[m] * ws[n];
      if (bias) v += bias[n];
      v = act8(v, act);
      if constexpr (sizeof(T) == 2) y[o] = __float2bfloat16(v);
      else y[o] = v;
    }
  }
}

// C [R][S] = sum over t of A(r, t) B(t, s), 32 x 32 tiles through shared memory
template <class T, class FA, class FB>
__global__ void __launch_bounds__(256) bwd_gemm_kernel(FA a, FB b, T* c, long long R, long long S, long long L) {
  __shared__ float sa[32][33], sb[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long r0 = static_cast<long long>(blockIdx.y) * 32, s0 = static_cast<long long>(blockIdx.x) * 32;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (long long t0 = 0; t0 < L; t0 += 32) {
    for (int i = 0; i < 4; ++i) {
      const int j = ty + 8 * i;
      sa[j][tx] = (r0 + j < R && t0 + tx < L) ? a(r0 + j, t0 + tx) : 0.f;
      sb[j][tx] = (t0 + j < L && s0 + tx < S) ? b(t0 + j, s0 + tx) : 0.f;
    }
    __syncthreads();
    for (int t = 0; t < 32; ++t)
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(sa[ty + 8 * i][t], sb[t][tx], acc[i]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const long long r = r0 + ty + 8 * i;
    if (r < R && s0 + tx < S) {
      if constexpr (sizeof(T) == 2) c[r * S + s0 + tx] = __float2bfloat16(acc[i]);
      else c[r * S + s0 + tx] = acc[i];
    }
  }
}
struct LoadB16 {
  const __nv_bfloat16* p; long long ld; bool t;
  __device__ float operator()(long long r, long long c) const { return __bfloat162float(t ? p[c * ld + r] : p[r * ld + c]); }
};
struct LoadQ8 {
  const int8_t* q; const float* s; long long ld;
  __device__ float operator()(long long r, long long c) const { return __bfloat162float(__float2bfloat16(q[r * ld + c] * s[r])); }
};
__global__ void __launch_bounds__(256) colsum_kernel(const __nv_bfloat16* __restrict__ g, float* __restrict__ out, long long M, int N) {
  const int n = blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= N) return;
  float acc = 0.f;
  for (long long m = 0; m < M; ++m) acc += __bfloat162float(g[m * N + n]);
  out[n] = acc;
}

}  // namespace
}  // namespace gb

using namespace gb;

extern "C" {

int grilly_linear_q8(grilly_ctx* ctx, const void* xq, const float* xs, const void* wq, const float* ws, const float* bias, void* y,
                     long long M, int N, int K, long long ldx, long long ldw, int act, int flags) {
  return rows8_entry(ctx, [&]() -> int {
    if (int rc = rows8_check(ctx, "linear_q8: x", xq, xs, M, K, ldx)) return rc;
    if (int rc = rows8_check(ctx, "linear_q8: weights", wq, ws, N, K, ldw)) return rc;
    if (N < 1) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "linear_q8: N must be positive");
    if (K > 131071) return set_error(ctx, GRILLY_ERR_UNSUPPORTED, "linear_q8: more than 131071 features can overflow the 32-bit sums");
    if (act < GRILLY_ACT_NONE || act > GRILLY_ACT_RELU) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "linear_q8: unknown activation");
    if (M == 0) return GRILLY_OK;
    if (!y) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "linear_q8: null output");
    const int grid = static_cast<int>(std::min<long long>((M * N + 7) / 8, ctx->num_sms * 8ll));
    if (flags & GRILLY_FLAG_OUT_BF16)
      linear_q8_kernel<<<grid, 256, 0, ctx->stream>>>(static_cast<const int8_t*>(xq), xs, static_cast<const int8_t*>(wq), ws, bias, static_cast<__nv_bfloat16*>(y), M, N, K, ldx, ldw, act);
    else
      linear_q8_kernel<<<grid, 256, 0, ctx->stream>>>(static_cast<const int8_t*>(xq), xs, static_cast<const int8_t*>(wq), ws, bias, static_cast<float*>(y), M, N, K, ldx, ldw, act);
    ctx->launches++;
    GB_CUDA_CHECK(ctx, cudaGetLastError());
    return GRILLY_OK;
  });
}

int grilly_linear_backward_q8(grilly_ctx* ctx, const void* go, const void* xq, const float* xs, const void* w, void* gx, void* gw, float* gbias,
                              long long M, int N, int K, long long ldx, int flags) {
  return rows8_entry(ctx, [&]() -> int {
    if (int rc = rows8_check(ctx, "linear_backward_q8: x", xq, xs, M, K, ldx)) return rc;
    if (N < 1) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "linear_backward_q8: N must be positive");
    const bool bf16 = flags & GRILLY_FLAG_OUT_BF16;
    if (M > 0 && !go) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "linear_backward_q8: null gradient");
    if (gx && !w) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "linear_backward_q8: grad_x needs the weights");
    const __nv_bfloat16* g = static_cast<const __nv_bfloat16*>(go);
    if (M == 0) {
      if (gw) GB_CUDA_CHECK(ctx, cudaMemsetAsync(gw, 0, static_cast<size_t>(N) * K * (bf16 ? 2 : 4), ctx->stream));
      if (gbias) GB_CUDA_CHECK(ctx, cudaMemsetAsync(gbias, 0, sizeof(float) * N, ctx->stream));
      return GRILLY_OK;
    }
    if (gx) {
      const dim3 grid((K + 31) / 32, static_cast<unsigned>((M + 31) / 32));
      LoadB16 a{g, N, false}, b{static_cast<const __nv_bfloat16*>(w), K, false};
      if (bf16) bwd_gemm_kernel<<<grid, 256, 0, ctx->stream>>>(a, b, static_cast<__nv_bfloat16*>(gx), M, K, N);
      else bwd_gemm_kernel<<<grid, 256, 0, ctx->stream>>>(a, b, static_cast<float*>(gx), M, K, N);
      ctx->launches++;
    }
    if (gw) {
      const dim3 grid((K + 31) / 32, (N + 31) / 32);
      LoadB16 a{g, N, true};
      LoadQ8 b{static_cast<const int8_t*>(xq), xs, ldx};
      if (bf16) bwd_gemm_kernel<<<grid, 256, 0, ctx->stream>>>(a, b, static_cast<__nv_bfloat16*>(gw), N, K, M);
      else bwd_gemm_kernel<<<grid, 256, 0, ctx->stream>>>(a, b, static_cast<float*>(gw), N, K, M);
      ctx->launches++;
    }
    if (gbias) {
      colsum_kernel<<<(N + 255) / 256, 256, 0, ctx->stream>>>(g, gbias, M, N);
      ctx->launches++;
    }
    GB_CUDA_CHECK(ctx, cudaGetLastError());
    return GRILLY_OK;
  });
}

}  // extern "C"
