// Rows in 8 bits: quantise, read back, RMSNorm with the residual's addition into 8-bit rows, and that norm's backward
// pass from the 8-bit checkpoint of its input. The definitions stand with the entry points in include/grilly_b200.h.
#include "rows8.h"
#include <cuda_bf16.h>
#include <algorithm>

namespace gb {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint32_t warp_max(uint32_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <class T> __device__ __forceinline__ float load_f(const T* p);
template <> __device__ __forceinline__ float load_f<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float load_f<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

// |x| as bits: non-negative floats order like their bits, an infinity is above every finite number and a NaN above that,
// so one integer maximum finds the largest magnitude and whether the row has a value that is not finite.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
constexpr uint32_t INF_BITS = 0x7f800000u;

__device__ __forceinline__ float row_scale(uint32_t amax_bits) {
  return amax_bits >= INF_BITS ? __uint_as_float(0x7fffffffu) : fmaxf(__uint_as_float(amax_bits) / 127.f, ROWS8_TINY);
}
// x / scale rounded to the nearest integer; a NaN (rows with scale NaN) converts to 0
__device__ __forceinline__ int8_t quant(float x, float inv) { return static_cast<int8_t>(__float2int_rn(x * inv)); }

// One warp per row, the row read twice: once for its largest magnitude, once to be written.
template <class T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* x, int8_t* q, float* scale, long long rows, int F, long long ld) {
  const int lane = threadIdx.x & 31;
  const long long step = static_cast<long long>(gridDim.x) * 8;
  for (long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); row < rows; row += step) {
    const T* xp = x + row * F;
    uint32_t m = 0;
    for (int i = lane; i < F; i += 32) m = max(m, abs_bits(load_f(xp + i)));
    const float s = row_scale(warp_max(m));
    const float inv = 1.f / s;
    int8_t* qp = q + row * ld;
    for (int i = lane; i < ld; i += 32) qp[i] = i < F ? quant(load_f(xp + i), inv) : int8_t(0);
    if (lane == 0) scale[row] = s;
  }
}

template <class T>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, T* y,
                                                              long long rows, int F, long long ld) {
  const int lane = threadIdx.x & 31;
  const long long step = static_cast<long long>(gridDim.x) * 8;
  for (long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); row < rows; row += step) {
    const float s = scale[row];
    for (int i = lane; i < F; i += 32) store_f(y + row * F + i, static_cast<float>(q[row * ld + i]) * s);
  }
}

struct NormQ8Args {
  const void* x;
  const void* residual;
  const float* gamma;
  void* h;
  int8_t* yq;
  float* ys;
  int8_t* hq;
  float* hs;
  float* rstd;
  long long rows, ld;
  int F;
  float eps;
};

// One reduction serves both outputs: the largest |h gamma| times rstd is the largest |y|, so sum h^2, max |h gamma| and
// max |h| are taken together and nothing waits for rstd.
template <class T>
__global__ void __launch_bounds__(256) rmsnorm_q8_kernel(const NormQ8Args a) {
  const int lane = threadIdx.x & 31;
  const long long step = static_cast<long long>(gridDim.x) * 8;
  for (long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); row < a.rows; row += step) {
    const T* xp = static_cast<const T*>(a.x) + row * a.F;
    const T* rp = a.residual ? static_cast<const T*>(a.residual) + row * a.F : nullptr;
    T* hp = a.h ? static_cast<T*>(a.h) + row * a.F : nullptr;
    float sq = 0.f;
    uint32_t my = 0, mh = 0;
    for (int i = lane; i < a.F; i += 32) {
      const float h = load_f(xp + i) + (rp ? load_f(rp + i) : 0.f);
      sq = fmaf(h, h, sq);
      my = max(my, abs_bits(h * (a.gamma ? a.gamma[i] : 1.f)));
      mh = max(mh, abs_bits(h));
    }
    sq = warp_sum(sq);
    my = warp_max(my);
    mh = warp_max(mh);
    const bool bad = abs_bits(sq) >= INF_BITS || my >= INF_BITS;
    const float rstd = bad ? __uint_as_float(0x7fffffffu) : __frsqrt_rn(sq / static_cast<float>(a.F) + a.eps);
    const float ys = bad ? __uint_as_float(0x7fffffffu) : row_scale(abs_bits(__uint_as_float(my) * rstd));
    const float hs = bad ? __uint_as_float(0x7fffffffu) : row_scale(mh);
    const float yi = 1.f / ys, hi = 1.f / hs;
    for (int i = lane; i < a.ld; i += 32) {
      float h = 0.f;
      if (i < a.F) {
        h = load_f(xp + i) + (rp ? load_f(rp + i) : 0.f);
        if (hp) store_f(hp + i, h);
      }
      a.yq[row * a.ld + i] = quant(h * rstd * ((a.gamma && i < a.F) ? a.gamma[i] : 1.f), yi);
      if (a.hq) a.hq[row * a.ld + i] = quant(h, hi);
    }
    if (lane == 0) {
      a.ys[row] = ys;
      if (a.hq) a.hs[row] = hs;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
}

struct NormBwdQ8Args {
  const void* go;
  const int8_t* hq;
  const float* hs;
  const float* rstd;
  const float* gamma;
  const void* gr;
  void* gh;
  float* partial;     // [blocks][F], or null
  long long rows, ld;
  int F;
};

template <class T>
__global__ void __launch_bounds__(256) rmsnorm_bwd_rows_kernel(const NormBwdQ8Args a) {
  const int lane = threadIdx.x & 31;
  const long long step = static_cast<long long>(gridDim.x) * 8;
  for (long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); row < a.rows; row += step) {
    const T* gp = static_cast<const T*>(a.go) + row * a.F;
    const T* rp = a.gr ? static_cast<const T*>(a.gr) + row * a.F : nullptr;
    T* op = static_cast<T*>(a.gh) + row * a.F;
    const int8_t* qp = a.hq + row * a.ld;
    const float rstd = a.rstd[row];
    const float s = a.hs[row] * rstd;
    float dot = 0.f;
    for (int i = lane; i < a.F; i += 32) dot = fmaf(load_f(gp + i) * (a.gamma ? a.gamma[i] : 1.f), qp[i] * s, dot);
    dot = warp_sum(dot) / static_cast<float>(a.F);
    for (int i = lane; i < a.F; i += 32) {
      const float g = load_f(gp + i) * (a.gamma ? a.gamma[i] : 1.f);
      store_f(op + i, rstd * (g - qp[i] * s * dot) + (rp ? load_f(rp + i) : 0.f));
    }
  }
}
template <class T>
__global__ void __launch_bounds__(256) rmsnorm_bwd_cols_kernel(const NormBwdQ8Args a, long long rows_per_block) {
  const long long r0 = static_cast<long long>(blockIdx.x) * rows_per_block;
  const long long r1 = min(a.rows, r0 + rows_per_block);
  for (int f = threadIdx.x; f < a.F; f += blockDim.x) {
    float acc = 0.f;
    for (long long r = r0; r < r1; ++r)
      acc = fmaf(load_f(static_cast<const T*>(a.go) + r * a.F + f), a.hq[r * a.ld + f] * (a.hs[r] * a.rstd[r]), acc);
    a.partial[static_cast<long long>(blockIdx.x) * a.F + f] = acc;
  }
}
__global__ void __launch_bounds__(256) sum_partials_kernel(const float* __restrict__ partial, float* __restrict__ out, int blocks, int F) {
  const int f = blockIdx.x * blockDim.x + threadIdx.x;
  if (f >= F) return;
  float acc = 0.f;
  for (int b = 0; b < blocks; ++b) acc += partial[static_cast<long long>(b) * F + f];
  out[f] = acc;
}

int row_grid(grilly_ctx* ctx, long long rows) { return static_cast<int>(std::min<long long>((rows + 7) / 8, ctx->num_sms * 8ll)); }

int done(grilly_ctx* ctx, int prof) {
  prof_end(ctx, prof);
  ctx->launches++;
  GB_CUDA_CHECK(ctx, cudaGetLastError());
  return GRILLY_OK;
}

}  // namespace
}  // namespace gb

using namespace gb;

extern "C" {

int grilly_quantize_rows(grilly_ctx* ctx, const void* x, void* q, float* scale, long long rows, int features, long long ld, int flags) {
  return rows8_entry(ctx, [&]() -> int {
    if (int rc = rows8_check(ctx, "quantize_rows", q, scale, rows, features, ld)) return rc;
    if (rows == 0) return GRILLY_OK;
    if (!x) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "quantize_rows: null input");
    const bool bf16 = flags & GRILLY_FLAG_IN_BF16;
    const int pi = prof_begin(ctx, PROF_NORM, 2.0 * rows * features, static_cast<double>(rows) * features * (bf16 ? 3 : 5) + 4.0 * rows);
    if (bf16) quantize_rows_kernel<<<row_grid(ctx, rows), 256, 0, ctx->stream>>>(static_cast<const __nv_bfloat16*>(x), static_cast<int8_t*>(q), scale, rows, features, ld);
    else quantize_rows_kernel<<<row_grid(ctx, rows), 256, 0, ctx->stream>>>(static_cast<const float*>(x), static_cast<int8_t*>(q), scale, rows, features, ld);
    return done(ctx, pi);
  });
}

int grilly_dequantize_rows(grilly_ctx* ctx, const void* q, const float* scale, void* y, long long rows, int features, long long ld, int flags) {
  return rows8_entry(ctx, [&]() -> int {
    if (int rc = rows8_check(ctx, "dequantize_rows", q, scale, rows, features, ld)) return rc;
    if (rows == 0) return GRILLY_OK;
    if (!y) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "dequantize_rows: null output");
    const bool bf16 = flags & GRILLY_FLAG_OUT_BF16;
    const int pi = prof_begin(ctx, PROF_NORM, 1.0 * rows * features, static_cast<double>(rows) * features * (bf16 ? 3 : 5) + 4.0 * rows);
    if (bf16) dequantize_rows_kernel<<<row_grid(ctx, rows), 256, 0, ctx->stream>>>(static_cast<const int8_t*>(q), scale, static_cast<__nv_bfloat16*>(y), rows, features, ld);
    else dequantize_rows_kernel<<<row_grid(ctx, rows), 256, 0, ctx->stream>>>(static_cast<const int8_t*>(q), scale, static_cast<float*>(y), rows, features, ld);
    return done(ctx, pi);
  });
}

int grilly_rmsnorm_residual_q8(grilly_ctx* ctx, const void* x, const void* residual, const float* gamma, void* h, void* y_q, float* y_scale,
                               void* h_q, float* h_scale, float* rstd, long long rows, int features, long long ld, float eps, int flags) {
  return rows8_entry(ctx, [&]() -> int {
    if (int rc = rows8_check(ctx, "rmsnorm_residual_q8", y_q, y_scale, rows, features, ld)) return rc;
    if (!h_q != !h_scale) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "rmsnorm_residual_q8: h_q and h_scale go together");
    if (reinterpret_cast<uintptr_t>(h_q) & 15) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "rmsnorm_residual_q8: 8-bit rows must be 16-byte aligned");
    if (!(eps > 0.f) || eps > 3.4e38f) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "rmsnorm_residual_q8: eps must be positive and finite");
    if (rows == 0) return GRILLY_OK;
    if (!x) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "rmsnorm_residual_q8: null input");
    const bool bf16 = flags & GRILLY_FLAG_IN_BF16;
    NormQ8Args a{x, residual, gamma, h, static_cast<int8_t*>(y_q), y_scale, static_cast<int8_t*>(h_q), h_scale, rstd, rows, ld, features, eps};
    const double e = bf16 ? 2 : 4, n = static_cast<double>(rows) * features;
    const int pi = prof_begin(ctx, PROF_NORM, 8.0 * n, n * (e * (1 + (residual ? 1 : 0) + (h ? 1 : 0)) + 1 + (h_q ? 1 : 0)) + 4.0 * features + 12.0 * rows);
    if (bf16) rmsnorm_q8_kernel<__nv_bfloat16><<<row_grid(ctx, rows), 256, 0, ctx->stream>>>(a);
    else rmsnorm_q8_kernel<float><<<row_grid(ctx, rows), 256, 0, ctx->stream>>>(a);
    return done(ctx, pi);
  });
}

int grilly_rmsnorm_backward_q8(grilly_ctx* ctx, const void* go, const void* h_q, const float* h_scale, const float* rstd, const float* gamma,
                               const void* grad_residual, void* grad_h, float* grad_gamma, long long rows, int features, long long ld, int flags) {
  return rows8_entry(ctx, [&]() -> int {
    if (int rc = rows8_check(ctx, "rmsnorm_backward_q8", h_q, h_scale, rows, features, ld)) return rc;
    if (rows == 0) {
      if (grad_gamma) GB_CUDA_CHECK(ctx, cudaMemsetAsync(grad_gamma, 0, sizeof(float) * features, ctx->stream));
      return GRILLY_OK;
    }
    if (!go || !rstd || !grad_h) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "rmsnorm_backward_q8: null operand");
    const bool bf16 = flags & GRILLY_FLAG_IN_BF16;
    NormBwdQ8Args a{go, static_cast<const int8_t*>(h_q), h_scale, rstd, gamma, grad_residual, grad_h, nullptr, rows, ld, features};
    Rows8Scratch scratch(ctx);
    int blocks = 0;
    if (grad_gamma) {
      blocks = static_cast<int>(std::min<long long>((rows + 31) / 32, ctx->num_sms));
      if (int rc = scratch.take(sizeof(float) * blocks * static_cast<size_t>(features))) return rc;
      a.partial = static_cast<float*>(scratch.p);
      // before grad_h is written: it may be grad_out
      const long long per = (rows + blocks - 1) / blocks;
      if (bf16) rmsnorm_bwd_cols_kernel<__nv_bfloat16><<<blocks, 256, 0, ctx->stream>>>(a, per);
      else rmsnorm_bwd_cols_kernel<float><<<blocks, 256, 0, ctx->stream>>>(a, per);
      ctx->launches++;
      sum_partials_kernel<<<(features + 255) / 256, 256, 0, ctx->stream>>>(a.partial, grad_gamma, blocks, features);
      ctx->launches++;
    }
    const double e = bf16 ? 2 : 4, n = static_cast<double>(rows) * features;
    const int pi = prof_begin(ctx, PROF_NORM, 10.0 * n, n * (e * (2 + (grad_residual ? 1 : 0)) + 1) + 8.0 * features + 8.0 * rows);
    if (bf16) rmsnorm_bwd_rows_kernel<__nv_bfloat16><<<row_grid(ctx, rows), 256, 0, ctx->stream>>>(a);
    else rmsnorm_bwd_rows_kernel<float><<<row_grid(ctx, rows), 256, 0, ctx->stream>>>(a);
    return done(ctx, pi);
  });
}

}  // extern "C"
