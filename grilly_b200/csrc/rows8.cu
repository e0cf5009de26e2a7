// Rows in 8 bits: quantise, read back, RMSNorm with the residual's addition into 8-bit rows, and that norm's backward
// pass from the 8-bit checkpoint of its input. The definitions stand with the entry points in include/grilly_b200.h.
//
// All of them are bound by HBM: a row is read once into the registers of a group of threads (a warp, or a block of up to
// 512 or 1024 threads; at most PER_THREAD values each), reduced once, and written once. Loads and stores are 16 bytes where the
// row length and the pointers allow it (fp32: 4 values, bf16: 8), else one value at a time with neighbouring lanes on
// neighbouring values.
#include "rows8.h"
#include "rows8_sum.cuh"
#include <cuda_bf16.h>
#include <algorithm>
#include <initializer_list>

namespace gb {
namespace {

constexpr int PER_THREAD = 32;         // values of a row per thread, forward kernels
constexpr int PER_THREAD_BWD = 16;     // backward: a thread also keeps its columns' gradient sums
constexpr uint32_t FULL = 0xffffffffu;
constexpr uint32_t INF_BITS = 0x7f800000u;
#define ROWS8_NAN __uint_as_float(0x7fffffffu)

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(FULL, v); }

// ---- VEC values of type T at p (16 bytes, or one value)
__device__ __forceinline__ void load_vec(const float* p, float (&v)[4]) {
  const float4 t = *reinterpret_cast<const float4*>(p);
  v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
}
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 t = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load_vec(const float* p, float (&v)[1]) { v[0] = *p; }
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, float (&v)[1]) { v[0] = __bfloat162float(*p); }
__device__ __forceinline__ void store_vec(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7]));
}
__device__ __forceinline__ void store_vec(float* p, const float (&v)[1]) { *p = v[0]; }
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[1]) { *p = __float2bfloat16(v[0]); }
// VEC fp32 parameters of the columns (1 where there are none)
template <int VEC>
__device__ __forceinline__ void load_gamma(const float* gamma, int col, float (&g)[VEC]) {
  if (!gamma) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) g[j] = 1.f;
  } else if constexpr (VEC == 1) {
    g[0] = __ldg(gamma + col);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 4) {
      const float4 t = __ldg(reinterpret_cast<const float4*>(gamma + col + j));
      g[j] = t.x; g[j + 1] = t.y; g[j + 2] = t.z; g[j + 3] = t.w;
    }
  }
}

// |x| as bits: non-negative floats order like their bits, an infinity is above every finite number and a NaN above that,
// so one integer maximum finds the largest magnitude and whether the row has a value that is not finite.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// max(amax / 127, 2^-126) or NaN. The quotient is the product with the rounded 1 / 127 and one correction by its remainder
// (Markstein), the correctly rounded one for every finite amax that is not clamped (checked over all significands).
__device__ __forceinline__ float row_scale(uint32_t amax_bits) {
  const float a = __uint_as_float(amax_bits), r = 1.f / 127.f, q = a * r;
  return amax_bits >= INF_BITS ? ROWS8_NAN : fmaxf(fmaf(fmaf(-127.f, q, a), r, q), ROWS8_TINY);
}
// 1 / scale to 1 ulp: it only decides values next to a tie. Scales lie in [2^-126, 2^121], where the approximation holds.
__device__ __forceinline__ float row_inverse(float scale) { return __fdividef(1.f, scale); }
// x * inv rounded to the nearest integer (ties to even), in the low byte: adding 1.5 * 2^23 leaves no fraction bits, and
// one fused multiply-add rounds once. Four bytes come out of three byte permutes; conversions would run at a quarter rate.
__device__ __forceinline__ uint32_t round_byte(float x, float inv) { return __float_as_uint(fmaf(x, inv, 12582912.f)); }
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// keep: all ones, or zero for a row that is not finite
__device__ __forceinline__ void store_q(int8_t* p, const float (&v)[8], float inv, uint32_t keep) {
  *reinterpret_cast<uint2*>(p) = make_uint2(
      pack4(round_byte(v[0], inv), round_byte(v[1], inv), round_byte(v[2], inv), round_byte(v[3], inv)) & keep,
      pack4(round_byte(v[4], inv), round_byte(v[5], inv), round_byte(v[6], inv), round_byte(v[7], inv)) & keep);
}
__device__ __forceinline__ void store_q(int8_t* p, const float (&v)[4], float inv, uint32_t keep) {
  *reinterpret_cast<uint32_t*>(p) = pack4(round_byte(v[0], inv), round_byte(v[1], inv), round_byte(v[2], inv), round_byte(v[3], inv)) & keep;
}
__device__ __forceinline__ void store_q(int8_t* p, const float (&v)[1], float inv, uint32_t keep) { *p = static_cast<int8_t>(round_byte(v[0], inv) & keep); }
// four signed bytes as floats: byte + 128 below the bits of 2^23, then the offset taken off; exact
__device__ __forceinline__ void unpack4(uint32_t w, float* v) {
  w ^= 0x80808080u;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + j)) - 8388736.f;
}
__device__ __forceinline__ void load_q(const int8_t* p, float (&v)[8]) {
  const uint2 t = *reinterpret_cast<const uint2*>(p);
  unpack4(t.x, v);
  unpack4(t.y, v + 4);
}
__device__ __forceinline__ void load_q(const int8_t* p, float (&v)[4]) { unpack4(*reinterpret_cast<const uint32_t*>(p), v); }
__device__ __forceinline__ void load_q(const int8_t* p, float (&v)[1]) { v[0] = static_cast<float>(*p); }

// A row's threads: a warp (eight rows per block of 256) or the whole block.
template <bool kWarp>
struct Group {
  long long row, step;
  int tid, size;
  __device__ Group() {
    if constexpr (kWarp) {
      row = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
      step = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
      tid = threadIdx.x & 31;
      size = 32;
    } else {
      row = blockIdx.x;
      step = gridDim.x;
      tid = threadIdx.x;
      size = blockDim.x;
    }
  }
};
struct RowStats {
  float sq;
  uint32_t my, mh;
};
// Over the group. `red` holds one entry per warp; a block calls it again only after its own __syncthreads.
template <bool kWarp, bool kSum, bool kTwo>
__device__ __forceinline__ RowStats group_reduce(RowStats s, RowStats* red) {
  if constexpr (kSum) s.sq = warp_sum(s.sq);
  s.mh = warp_max(s.mh);
  if constexpr (kTwo) s.my = warp_max(s.my);
  if constexpr (!kWarp) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    s = lane < warps ? red[lane] : RowStats{0.f, 0u, 0u};
    if constexpr (kSum) s.sq = warp_sum(s.sq);
    s.mh = warp_max(s.mh);
    if constexpr (kTwo) s.my = warp_max(s.my);
  }
  return s;
}

// ---------------------------------------------------------------- quantise
template <class T, int VEC, bool kWarp>
__global__ void __launch_bounds__(kWarp ? 256 : 512) quantize_rows_kernel(const T* x, int8_t* q, float* scale, long long rows, int F, long long ld) {
  constexpr int NV = PER_THREAD / VEC;
  __shared__ RowStats red[32];
  const Group<kWarp> g;
  for (long long row = g.row; row < rows; row += g.step) {
    const T* xp = x + row * F;
    float v[NV][VEC];
    RowStats s{0.f, 0u, 0u};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (g.tid + i * g.size) * VEC;
      if (c < F) load_vec(xp + c, v[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((g.tid + i * g.size) * VEC < F) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) s.mh = max(s.mh, abs_bits(v[i][j]));
      }
    }
    s = group_reduce<kWarp, false, false>(s, red);
    const float sc = row_scale(s.mh), inv = row_inverse(sc);
    const uint32_t keep = s.mh >= INF_BITS ? 0u : FULL;
    int8_t* qp = q + row * ld;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (g.tid + i * g.size) * VEC;
      if (c < F) store_q(qp + c, v[i], inv, keep);
    }
    for (long long c = F + g.tid; c < ld; c += g.size) qp[c] = 0;
    if (g.tid == 0) scale[row] = sc;
    if constexpr (!kWarp) __syncthreads();
  }
}
// Rows too long for a block's registers: read twice.
template <class T>
__global__ void __launch_bounds__(1024) quantize_long_rows_kernel(const T* x, int8_t* q, float* scale, long long rows, int F, long long ld) {
  __shared__ RowStats red[32];
  const Group<false> g;
  for (long long row = g.row; row < rows; row += g.step) {
    const T* xp = x + row * F;
    RowStats s{0.f, 0u, 0u};
    float v[1];
    for (int c = g.tid; c < F; c += g.size) {
      load_vec(xp + c, v);
      s.mh = max(s.mh, abs_bits(v[0]));
    }
    s = group_reduce<false, false, false>(s, red);
    const float sc = row_scale(s.mh), inv = row_inverse(sc);
    const uint32_t keep = s.mh >= INF_BITS ? 0u : FULL;
    for (long long c = g.tid; c < ld; c += g.size) {
      v[0] = 0.f;
      if (c < F) load_vec(xp + c, v);
      store_q(q + row * ld + c, v, inv, keep);
    }
    if (g.tid == 0) scale[row] = sc;
    __syncthreads();
  }
}

// ---------------------------------------------------------------- read back
// 16 values per thread; the caller made sure that the vectors of all rows can be counted in 32 bits.
template <class T>
__global__ void __launch_bounds__(256) dequantize_vec_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, T* __restrict__ y,
                                                             uint32_t vectors, uint32_t per_row, long long ld) {
  constexpr int VEC = 16 / sizeof(T);
  for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < vectors; i += gridDim.x * 256u) {
    const uint32_t row = i / per_row, c = (i - row * per_row) * 16;
    const uint4 w = *reinterpret_cast<const uint4*>(q + row * ld + c);
    const float s = __ldg(scale + row);
    float v[16];
    unpack4(w.x, v); unpack4(w.y, v + 4); unpack4(w.z, v + 8); unpack4(w.w, v + 12);
    T* yp = y + (static_cast<long long>(row) * per_row * 16 + c);
#pragma unroll
    for (int k = 0; k < 16; k += VEC) {
      float o[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) o[j] = v[k + j] * s;
      store_vec(yp + k, o);
    }
  }
}
// Any row length: one warp per row.
template <class T>
__global__ void __launch_bounds__(256) dequantize_any_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, T* __restrict__ y,
                                                             long long rows, int F, long long ld) {
  const Group<true> g;
  for (long long row = g.row; row < rows; row += g.step) {
    const float s = __ldg(scale + row);
#pragma unroll 8
    for (int c = g.tid; c < F; c += 32) {
      const float v[1] = {static_cast<float>(q[row * ld + c]) * s};
      store_vec(y + row * F + c, v);
    }
  }
}

// ---------------------------------------------------------------- RMSNorm with the residual's addition
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
struct NormScales {
  float rstd, ys, hs, yi, hi;
  uint32_t keep;
};
__device__ __forceinline__ NormScales norm_scales(const RowStats& s, float inv_f, float eps) {
  NormScales r;
  const bool bad = abs_bits(s.sq) >= INF_BITS || s.my >= INF_BITS;
  r.keep = bad ? 0u : FULL;
  const float var = s.sq * inv_f + eps;
  float t = rsqrtf(var);                       // within 2 ulp; one Newton step brings it to the rounding of 1 / sqrt
  t = fmaf(t, fmaf(-0.5f * var * t, t, 0.5f), t);
  r.rstd = bad ? ROWS8_NAN : t;
  r.ys = bad ? ROWS8_NAN : row_scale(abs_bits(__uint_as_float(s.my) * r.rstd));
  r.hs = bad ? ROWS8_NAN : row_scale(s.mh);
  r.yi = row_inverse(r.ys);
  r.hi = row_inverse(r.hs);
  return r;
}
__device__ __forceinline__ void norm_row_done(const NormQ8Args& a, const NormScales& r, long long row) {
  a.ys[row] = r.ys;
  if (a.hq) a.hs[row] = r.hs;
  if (a.rstd) a.rstd[row] = r.rstd;
}

// One reduction serves both outputs: the largest |h gamma| times rstd is the largest |y|, so sum h^2, max |h gamma| and
// max |h| are taken together and nothing waits for rstd. h is written after the whole row has been read (in place).
template <class T, int VEC, bool kWarp>
__global__ void __launch_bounds__(kWarp ? 256 : 512) rmsnorm_q8_kernel(const NormQ8Args a) {
  constexpr int NV = PER_THREAD / VEC;
  __shared__ RowStats red[32];
  const Group<kWarp> g;
  const int F = a.F;
  const float inv_f = 1.f / static_cast<float>(F);
  for (long long row = g.row; row < a.rows; row += g.step) {
    const T* xp = static_cast<const T*>(a.x) + row * F;
    const T* rp = a.residual ? static_cast<const T*>(a.residual) + row * F : nullptr;
    float h[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (g.tid + i * g.size) * VEC;
      if (c < F) load_vec(xp + c, h[i]);
    }
    if (rp) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (g.tid + i * g.size) * VEC;
        if (c < F) {
          float r[VEC];
          load_vec(rp + c, r);
#pragma unroll
          for (int j = 0; j < VEC; ++j) h[i][j] += r[j];
        }
      }
    }
    RowStats s{0.f, 0u, 0u};
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (g.tid + i * g.size) * VEC;
      if (c < F) {
        float gm[VEC];
        load_gamma(a.gamma, c, gm);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float& acc = sum[(i * VEC + j) & 3];
          acc = fmaf(h[i][j], h[i][j], acc);
          s.my = max(s.my, abs_bits(h[i][j] * gm[j]));
          s.mh = max(s.mh, abs_bits(h[i][j]));
        }
      }
    }
    s.sq = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    s = group_reduce<kWarp, true, true>(s, red);
    const NormScales r = norm_scales(s, inv_f, a.eps);
    T* hp = a.h ? static_cast<T*>(a.h) + row * F : nullptr;
    int8_t* yq = a.yq + row * a.ld;
    int8_t* hq = a.hq ? a.hq + row * a.ld : nullptr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (g.tid + i * g.size) * VEC;
      if (c < F) {
        if (hp) store_vec(hp + c, h[i]);
        if (hq) store_q(hq + c, h[i], r.hi, r.keep);
        float gm[VEC];
        load_gamma(a.gamma, c, gm);
#pragma unroll
        for (int j = 0; j < VEC; ++j) gm[j] *= h[i][j] * r.rstd;
        store_q(yq + c, gm, r.yi, r.keep);
      }
    }
    for (long long c = F + g.tid; c < a.ld; c += g.size) {
      yq[c] = 0;
      if (hq) hq[c] = 0;
    }
    if (g.tid == 0) norm_row_done(a, r, row);
    if constexpr (!kWarp) __syncthreads();
  }
}
// Rows too long for a block's registers: read twice, h written as it is read again.
template <class T>
__global__ void __launch_bounds__(1024) rmsnorm_q8_long_kernel(const NormQ8Args a) {
  __shared__ RowStats red[32];
  const Group<false> g;
  for (long long row = g.row; row < a.rows; row += g.step) {
    const T* xp = static_cast<const T*>(a.x) + row * a.F;
    const T* rp = a.residual ? static_cast<const T*>(a.residual) + row * a.F : nullptr;
    RowStats s{0.f, 0u, 0u};
    float h[1], r[1], gm[1];
    auto in = [&](int c) {
      load_vec(xp + c, h);
      if (rp) {
        load_vec(rp + c, r);
        h[0] += r[0];
      }
      load_gamma(a.gamma, c, gm);
    };
    for (int c = g.tid; c < a.F; c += g.size) {
      in(c);
      s.sq = fmaf(h[0], h[0], s.sq);
      s.my = max(s.my, abs_bits(h[0] * gm[0]));
      s.mh = max(s.mh, abs_bits(h[0]));
    }
    s = group_reduce<false, true, true>(s, red);
    const NormScales n = norm_scales(s, 1.f / static_cast<float>(a.F), a.eps);
    for (long long c = g.tid; c < a.ld; c += g.size) {
      h[0] = gm[0] = 0.f;
      if (c < a.F) {
        in(static_cast<int>(c));
        if (a.h) store_vec(static_cast<T*>(a.h) + row * a.F + c, h);
      }
      if (a.hq) store_q(a.hq + row * a.ld + c, h, n.hi, n.keep);
      gm[0] *= h[0] * n.rstd;
      store_q(a.yq + row * a.ld + c, gm, n.yi, n.keep);
    }
    if (g.tid == 0) norm_row_done(a, n, row);
    __syncthreads();
  }
}

// ---------------------------------------------------------------- backward pass of the norm
struct NormBwdQ8Args {
  const void* go;
  const int8_t* hq;
  const float* hs;
  const float* rstd;
  const float* gamma;
  const void* gr;
  void* gh;
  float* partial;     // [blocks][F] sums of grad_out * n over a block's rows, or null
  long long rows, ld;
  int F, group;       // threads per row
};

// A block walks rows with one group of threads per row (blockDim / group rows at a time). A thread keeps the same columns
// of every row it meets, so the gradient of gamma is summed in registers and leaves once per block; the blocks' sums are
// added by sum_partials_kernel in a fixed order. The whole row of grad_out and grad_residual is in registers before the
// first store (in place).
template <class T, int VEC, int MAX_THREADS>
__global__ void __launch_bounds__(MAX_THREADS) rmsnorm_bwd_kernel(const NormBwdQ8Args a) {
  constexpr int NV = PER_THREAD_BWD / VEC;
  extern __shared__ float columns[];               // [F], with partial
  __shared__ float red[2][32];
  const int F = a.F, G = a.group;
  const int groups = blockDim.x / G, which = threadIdx.x / G, tid = threadIdx.x - which * G;
  const int lane = threadIdx.x & 31, first_warp = which * (G >> 5), warps = G >> 5;
  const float inv_f = 1.f / static_cast<float>(F);
  float acc[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[i][j] = 0.f;
  int parity = 0;
  for (long long row = static_cast<long long>(blockIdx.x) * groups + which; row < a.rows; row += static_cast<long long>(gridDim.x) * groups, parity ^= 1) {
    const T* gp = static_cast<const T*>(a.go) + row * F;
    const T* rp = a.gr ? static_cast<const T*>(a.gr) + row * F : nullptr;
    const int8_t* qp = a.hq + row * a.ld;
    float g[NV][VEC], n[NV][VEC], r[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (tid + i * G) * VEC;
      if (c < F) {
        load_vec(gp + c, g[i]);
        load_q(qp + c, n[i]);
        if (rp) load_vec(rp + c, r[i]);
      }
    }
    const float rstd = a.rstd[row], s = a.hs[row] * rstd;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (tid + i * G) * VEC;
      if (c < F) {
        float gm[VEC];
        load_gamma(a.gamma, c, gm);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          n[i][j] *= s;
          acc[i][j] = fmaf(g[i][j], n[i][j], acc[i][j]);
          g[i][j] *= gm[j];
          dot = fmaf(g[i][j], n[i][j], dot);
        }
      }
    }
    dot = warp_sum(dot);
    if (warps > 1) {
      if (lane == 0) red[parity][threadIdx.x >> 5] = dot;
      // the group's own barrier; the other half of `red` is written before the next one, so one per row is enough
      asm volatile("bar.sync %0, %1;" ::"r"(which + 1), "r"(G) : "memory");
      dot = warp_sum(lane < warps ? red[parity][first_warp + lane] : 0.f);
    }
    dot *= inv_f;
    T* op = static_cast<T*>(a.gh) + row * F;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (tid + i * G) * VEC;
      if (c < F) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          g[i][j] = rstd * (g[i][j] - n[i][j] * dot);
          if (rp) g[i][j] += r[i][j];
        }
        store_vec(op + c, g[i]);
      }
    }
  }
  if (!a.partial) return;
  for (int w = 0; w < groups; ++w) {
    if (which == w) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (tid + i * G) * VEC;
        if (c < F) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) columns[c + j] = w == 0 ? acc[i][j] : columns[c + j] + acc[i][j];
        }
      }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < F; c += blockDim.x) a.partial[static_cast<long long>(blockIdx.x) * F + c] = columns[c];
}
// Rows too long for a block's registers: the rows in two passes, the columns by themselves before them (grad_h may be
// grad_out).
template <class T>
__global__ void __launch_bounds__(1024) rmsnorm_bwd_long_rows_kernel(const NormBwdQ8Args a) {
  __shared__ RowStats red[32];
  const Group<false> gr;
  for (long long row = gr.row; row < a.rows; row += gr.step) {
    const T* gp = static_cast<const T*>(a.go) + row * a.F;
    const T* rp = a.gr ? static_cast<const T*>(a.gr) + row * a.F : nullptr;
    T* op = static_cast<T*>(a.gh) + row * a.F;
    const int8_t* qp = a.hq + row * a.ld;
    const float rstd = a.rstd[row], s = a.hs[row] * rstd;
    RowStats st{0.f, 0u, 0u};
    float g[1], gm[1], r[1] = {0.f};
    for (int c = gr.tid; c < a.F; c += gr.size) {
      load_vec(gp + c, g);
      load_gamma(a.gamma, c, gm);
      st.sq = fmaf(g[0] * gm[0], static_cast<float>(qp[c]) * s, st.sq);
    }
    const float dot = group_reduce<false, true, false>(st, red).sq / static_cast<float>(a.F);
    for (int c = gr.tid; c < a.F; c += gr.size) {
      load_vec(gp + c, g);
      load_gamma(a.gamma, c, gm);
      if (rp) load_vec(rp + c, r);
      g[0] = rstd * (g[0] * gm[0] - static_cast<float>(qp[c]) * s * dot) + r[0];
      store_vec(op + c, g);
    }
    __syncthreads();
  }
}
template <class T>
__global__ void __launch_bounds__(256) rmsnorm_bwd_long_columns_kernel(const NormBwdQ8Args a, long long rows_per_block) {
  const long long r0 = static_cast<long long>(blockIdx.x) * rows_per_block;
  const long long r1 = min(a.rows, r0 + rows_per_block);
  for (int f = threadIdx.x; f < a.F; f += blockDim.x) {
    float acc = 0.f, g[1];
    for (long long r = r0; r < r1; ++r) {
      load_vec(static_cast<const T*>(a.go) + r * a.F + f, g);
      acc = fmaf(g[0], static_cast<float>(a.hq[r * a.ld + f]) * (a.hs[r] * a.rstd[r]), acc);
    }
    a.partial[static_cast<long long>(blockIdx.x) * a.F + f] = acc;
  }
}
// ---------------------------------------------------------------- launch shapes
bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  return true;
}
// Threads of a row, by its length alone: a row's sums have the same order, and its result the same bits, in every batch.
struct RowShape {
  bool warp;
  int threads;
  unsigned grid;
};
#ifndef PER_TARGET
#define PER_TARGET 32
#endif
RowShape row_shape(long long rows, int F) {
  if (F <= 32 * PER_THREAD) return {true, 256, static_cast<unsigned>(std::min<long long>((rows + 7) / 8, 1 << 20))};
  const int threads = std::min(512, (F + PER_TARGET - 1) / PER_TARGET);
  return {false, (threads + 31) / 32 * 32, static_cast<unsigned>(std::min<long long>(rows, 1 << 20))};
}
constexpr int LONGEST_ROW = 512 * PER_THREAD;
constexpr int LONGEST_ROW_BWD = 1024 * PER_THREAD_BWD;

template <class T>
void launch_quantize(grilly_ctx* ctx, const T* x, int8_t* q, float* scale, long long rows, int F, long long ld) {
  constexpr int VEC = 16 / sizeof(T);
  const cudaStream_t st = ctx->stream;
  if (F > LONGEST_ROW) {
    quantize_long_rows_kernel<<<static_cast<unsigned>(std::min<long long>(rows, 1 << 20)), 1024, 0, st>>>(x, q, scale, rows, F, ld);
    return;
  }
  const RowShape s = row_shape(rows, F);
  const bool vec = F % VEC == 0 && aligned16({x});
  if (s.warp) {
    if (vec) quantize_rows_kernel<T, VEC, true><<<s.grid, s.threads, 0, st>>>(x, q, scale, rows, F, ld);
    else quantize_rows_kernel<T, 1, true><<<s.grid, s.threads, 0, st>>>(x, q, scale, rows, F, ld);
  } else {
    if (vec) quantize_rows_kernel<T, VEC, false><<<s.grid, s.threads, 0, st>>>(x, q, scale, rows, F, ld);
    else quantize_rows_kernel<T, 1, false><<<s.grid, s.threads, 0, st>>>(x, q, scale, rows, F, ld);
  }
}

template <class T>
void launch_dequantize(grilly_ctx* ctx, const int8_t* q, const float* scale, T* y, long long rows, int F, long long ld) {
  const cudaStream_t st = ctx->stream;
  const long long vectors = rows * (F / 16);
  if (F % 16 == 0 && aligned16({y}) && vectors < (1ll << 31)) {
    const unsigned grid = static_cast<unsigned>(std::min<long long>((vectors + 255) / 256, ctx->num_sms * 32ll));
    dequantize_vec_kernel<T><<<grid, 256, 0, st>>>(q, scale, y, static_cast<uint32_t>(vectors), static_cast<uint32_t>(F / 16), ld);
  } else {
    dequantize_any_kernel<T><<<static_cast<unsigned>(std::min<long long>((rows + 7) / 8, 1 << 20)), 256, 0, st>>>(q, scale, y, rows, F, ld);
  }
}

template <class T>
void launch_rmsnorm(grilly_ctx* ctx, const NormQ8Args& a) {
  constexpr int VEC = 16 / sizeof(T);
  const cudaStream_t st = ctx->stream;
  if (a.F > LONGEST_ROW) {
    rmsnorm_q8_long_kernel<T><<<static_cast<unsigned>(std::min<long long>(a.rows, 1 << 20)), 1024, 0, st>>>(a);
    return;
  }
  const RowShape s = row_shape(a.rows, a.F);
  const bool vec = a.F % VEC == 0 && aligned16({a.x, a.residual, a.gamma, a.h});
  if (s.warp) {
    if (vec) rmsnorm_q8_kernel<T, VEC, true><<<s.grid, s.threads, 0, st>>>(a);
    else rmsnorm_q8_kernel<T, 1, true><<<s.grid, s.threads, 0, st>>>(a);
  } else {
    if (vec) rmsnorm_q8_kernel<T, VEC, false><<<s.grid, s.threads, 0, st>>>(a);
    else rmsnorm_q8_kernel<T, 1, false><<<s.grid, s.threads, 0, st>>>(a);
  }
}

template <class T, int VEC, int MAX_THREADS>
int launch_rmsnorm_bwd_vec(grilly_ctx* ctx, NormBwdQ8Args& a, float* grad_gamma) {
  auto kern = rmsnorm_bwd_kernel<T, VEC, MAX_THREADS>;
  a.group = ((a.F + PER_THREAD_BWD - 1) / PER_THREAD_BWD + 31) / 32 * 32;
  const int groups = std::max(1, 256 / a.group), threads = groups * a.group;
  const size_t smem = grad_gamma ? sizeof(float) * a.F : 0;
  const void* key = reinterpret_cast<const void*>(kern);
  if (!ctx->smem_attr_done.count(key)) {
    GB_CUDA_CHECK(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, LONGEST_ROW_BWD * 4));
    ctx->smem_attr_done.insert(key);
  }
  int per_sm = 0;
  GB_CUDA_CHECK(ctx, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem));
  const int blocks = static_cast<int>(std::min<long long>((a.rows + groups - 1) / groups, static_cast<long long>(ctx->num_sms) * std::max(1, per_sm)));
  Rows8Scratch scratch(ctx);
  if (grad_gamma) {
    if (int rc = scratch.take(sizeof(float) * blocks * static_cast<size_t>(a.F))) return rc;
    a.partial = static_cast<float*>(scratch.p);
  }
  kern<<<blocks, threads, smem, ctx->stream>>>(a);
  ctx->launches++;
  if (grad_gamma) {
    sum_partials_kernel<<<(a.F + 31) / 32, 512, 0, ctx->stream>>>(a.partial, grad_gamma, blocks, a.F);
    ctx->launches++;
  }
  GB_CUDA_CHECK(ctx, cudaGetLastError());
  return GRILLY_OK;
}
template <class T>
int launch_rmsnorm_bwd(grilly_ctx* ctx, NormBwdQ8Args& a, float* grad_gamma) {
  constexpr int VEC = 16 / sizeof(T);
  if (a.F <= LONGEST_ROW_BWD) {
    const bool vec = a.F % VEC == 0 && aligned16({a.go, a.gr, a.gh, a.gamma});
    // up to 512 threads per row there are registers for everything a thread holds; 1024 threads spill a little
    if (a.F <= 512 * PER_THREAD_BWD)
      return vec ? launch_rmsnorm_bwd_vec<T, VEC, 512>(ctx, a, grad_gamma) : launch_rmsnorm_bwd_vec<T, 1, 512>(ctx, a, grad_gamma);
    return vec ? launch_rmsnorm_bwd_vec<T, VEC, 1024>(ctx, a, grad_gamma) : launch_rmsnorm_bwd_vec<T, 1, 1024>(ctx, a, grad_gamma);
  }
  Rows8Scratch scratch(ctx);
  if (grad_gamma) {
    const int blocks = static_cast<int>(std::min<long long>((a.rows + 31) / 32, ctx->num_sms));
    const long long per = (a.rows + blocks - 1) / blocks;
    if (int rc = scratch.take(sizeof(float) * blocks * static_cast<size_t>(a.F))) return rc;
    a.partial = static_cast<float*>(scratch.p);
    rmsnorm_bwd_long_columns_kernel<T><<<blocks, 256, 0, ctx->stream>>>(a, per);
    sum_partials_kernel<<<(a.F + 31) / 32, 512, 0, ctx->stream>>>(a.partial, grad_gamma, blocks, a.F);
    ctx->launches += 2;
  }
  rmsnorm_bwd_long_rows_kernel<T><<<static_cast<unsigned>(std::min<long long>(a.rows, 1 << 20)), 1024, 0, ctx->stream>>>(a);
  ctx->launches++;
  GB_CUDA_CHECK(ctx, cudaGetLastError());
  return GRILLY_OK;
}

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
    if (bf16) launch_quantize(ctx, static_cast<const __nv_bfloat16*>(x), static_cast<int8_t*>(q), scale, rows, features, ld);
    else launch_quantize(ctx, static_cast<const float*>(x), static_cast<int8_t*>(q), scale, rows, features, ld);
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
    if (bf16) launch_dequantize(ctx, static_cast<const int8_t*>(q), scale, static_cast<__nv_bfloat16*>(y), rows, features, ld);
    else launch_dequantize(ctx, static_cast<const int8_t*>(q), scale, static_cast<float*>(y), rows, features, ld);
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
    if (bf16) launch_rmsnorm<__nv_bfloat16>(ctx, a);
    else launch_rmsnorm<float>(ctx, a);
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
    NormBwdQ8Args a{go, static_cast<const int8_t*>(h_q), h_scale, rstd, gamma, grad_residual, grad_h, nullptr, rows, ld, features, 0};
    const double e = bf16 ? 2 : 4, n = static_cast<double>(rows) * features;
    const int pi = prof_begin(ctx, PROF_NORM, 10.0 * n, n * (e * (2 + (grad_residual ? 1 : 0)) + 1) + 8.0 * features + 8.0 * rows);
    const int rc = bf16 ? launch_rmsnorm_bwd<__nv_bfloat16>(ctx, a, grad_gamma) : launch_rmsnorm_bwd<float>(ctx, a, grad_gamma);
    prof_end(ctx, pi);
    return rc;
  });
}

}  // extern "C"
