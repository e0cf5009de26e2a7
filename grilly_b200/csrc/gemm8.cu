// Matrix products over 8-bit rows: y = act(s_x s_w x_q W_q^T + b), and the backward pass of a linear layer whose saved
// input is in 8-bit rows. The definitions stand with the entry points in include/grilly_b200.h.
#include "rows8.h"
#include "rows8_sum.cuh"
#include "gemm8.cuh"
#include <algorithm>

namespace gb {
namespace {

// ---------------------------------------------------------------- few tokens: bound by reading the weights once
struct FewArgs {
  const int8_t* xq;
  const float* xs;
  const int8_t* wq;
  const float* ws;
  const float* bias;
  void* y;
  int M, N, K;
  long long ldx, ldw;
  int act, out_bf16;
};
constexpr int FEW_TOKENS = 32;

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the first n bytes of a 16-byte piece
__device__ __forceinline__ uint4 first_bytes(uint4 v, int n) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int left = n - 4 * i;
    if (left <= 0) w[i] = 0;
    else if (left < 4) w[i] &= (1u << (8 * left)) - 1u;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 features per block; its 8 warps walk K in pieces of 64. Both operands come straight from memory in 16-byte pieces: the
// sum over k does not care which k a lane calls its own, so lane t of four takes 16 consecutive bytes of a row and feeds
// them to two MMAs as if they were the fragment's columns, the same for weights and tokens. Rows past the end repeat the
// last one (their results are dropped); bytes past K are zeroed on the tokens' side. The warps' sums join in shared memory.
template <int NT>
__global__ void __launch_bounds__(256) linear_q8_few_kernel(const FewArgs a) {
  __shared__ int red[8][16][8 * NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int f0 = blockIdx.x * 16;
  const int8_t* w0 = a.wq + static_cast<long long>(min(f0 + g, a.N - 1)) * a.ldw + t * 16;
  const int8_t* w1 = a.wq + static_cast<long long>(min(f0 + g + 8, a.N - 1)) * a.ldw + t * 16;
  const int8_t* x[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) x[n] = a.xq + static_cast<long long>(min(n * 8 + g, a.M - 1)) * a.ldx + t * 16;
  int acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0;
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll 4
  for (int k = warp * 64; k < a.K; k += 8 * 64) {
    const int left = a.K - k - t * 16;         // bytes of this lane's piece inside the row
    uint4 p0 = zero, p1 = zero, q[NT];
    if (left > 0) {
      p0 = __ldg(reinterpret_cast<const uint4*>(w0 + k));
      p1 = __ldg(reinterpret_cast<const uint4*>(w1 + k));
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) q[n] = left > 0 ? __ldg(reinterpret_cast<const uint4*>(x[n] + k)) : zero;
    if (left < 16) {
#pragma unroll
      for (int n = 0; n < NT; ++n) q[n] = first_bytes(q[n], left);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      mma_s8(acc[n], p0.x, p1.x, p0.y, p1.y, q[n].x, q[n].y);
      mma_s8(acc[n], p0.z, p1.z, p0.w, p1.w, q[n].z, q[n].w);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    red[warp][g][8 * n + 2 * t] = acc[n][0];
    red[warp][g][8 * n + 2 * t + 1] = acc[n][1];
    red[warp][g + 8][8 * n + 2 * t] = acc[n][2];
    red[warp][g + 8][8 * n + 2 * t + 1] = acc[n][3];
  }
  __syncthreads();
  for (int o = threadIdx.x; o < 16 * 8 * NT; o += 256) {
    const int f = f0 + (o & 15), m = o >> 4;
    if (f >= a.N || m >= a.M) continue;
    int s = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += red[w][o & 15][m];
    const float v = gemm8_act(fmaf(static_cast<float>(s) * __ldg(a.xs + m), __ldg(a.ws + f), a.bias ? __ldg(a.bias + f) : 0.f), a.act);
    const long long at = static_cast<long long>(m) * a.N + f;
    if (a.out_bf16) static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16(v);
    else static_cast<float*>(a.y)[at] = v;
  }
}

// ---------------------------------------------------------------- operands of the backward pass
// q * scale rounded to bf16, rows of ld values (what lies past the features is never read as a column)
__global__ void __launch_bounds__(256) expand_rows_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, __nv_bfloat16* __restrict__ y,
                                                          long long pieces, int per_row) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < pieces; i += gridDim.x * 256ll) {
    const float s = __ldg(scale + i / per_row);
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(q) + i);
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
    uint32_t out[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t u = in[j] ^ 0x80808080u;
      float v[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) v[b] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + b)) - 8388736.f) * s;
      const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
      out[2 * j] = *reinterpret_cast<const uint32_t*>(&lo);
      out[2 * j + 1] = *reinterpret_cast<const uint32_t*>(&hi);
    }
    uint4* yp = reinterpret_cast<uint4*>(y) + 2 * i;
    yp[0] = make_uint4(out[0], out[1], out[2], out[3]);
    yp[1] = make_uint4(out[4], out[5], out[6], out[7]);
  }
}
// rows of n bf16 values to rows of ld values, for TMA, which wants rows on 16-byte boundaries
__global__ void __launch_bounds__(256) pitch_rows_kernel(const __nv_bfloat16* __restrict__ x, __nv_bfloat16* __restrict__ y, long long rows, int n, int ld) {
  const int lane = threadIdx.x & 31;
  for (long long row = blockIdx.x * 8ll + (threadIdx.x >> 5); row < rows; row += gridDim.x * 8ll) {
#pragma unroll 8
    for (int c = lane; c < n; c += 32) y[row * ld + c] = x[row * n + c];
  }
}
// partial[block][n] = sum over the block's rows. V columns per thread.
template <int V>
__global__ void __launch_bounds__(256) column_sums_kernel(const __nv_bfloat16* __restrict__ g, float* __restrict__ partial, long long M, int N, long long rows_per_block) {
  const int n = (blockIdx.x * 256 + threadIdx.x) * V;
  if (n >= N) return;
  const long long r0 = blockIdx.y * rows_per_block, r1 = min(M, r0 + rows_per_block);
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
#pragma unroll 8
  for (long long r = r0; r < r1; ++r) {
    if constexpr (V == 8) {
      const uint4 t = __ldg(reinterpret_cast<const uint4*>(g + r * N + n));
      const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[2 * j] += __uint_as_float(w[j] << 16);
        acc[2 * j + 1] += __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {
      acc[0] += __bfloat162float(g[r * N + n]);
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) partial[static_cast<long long>(blockIdx.y) * N + n + j] = acc[j];
}

// ---------------------------------------------------------------- launches
struct Operand {
  const void* p;
  long long ld;      // elements between rows
};

// C [M][N] of KIND over k; `a` and `b` as the kind reads them.
template <Gemm8Kind KIND>
int launch_gemm8(grilly_ctx* ctx, Operand oa, Operand ob, long long M, int N, long long k, Gemm8Args& g) {
  using Cfg = Gemm8Cfg;
  constexpr bool kInt8 = KIND == Gemm8Kind::Q8;
  constexpr int BK = kInt8 ? 128 : 64;
  if (M > 0x7fffff00ll || k > 0x7fffff00ll || N > 0x7fffff00) return set_error(ctx, GRILLY_ERR_UNSUPPORTED, "8-bit rows: more than 2^31 - 256 rows");
  CUtensorMap ta, tb;
  int rc;
  if (kInt8) {
    if ((rc = get_tmap_2d(ctx, TM_U8, oa.p, k, M, oa.ld, BK, 128, &ta))) return rc;
    if ((rc = get_tmap_2d(ctx, TM_U8, ob.p, k, N, ob.ld, BK, 128, &tb))) return rc;
  } else {
    if (KIND == Gemm8Kind::WGRAD) rc = get_tmap_2d(ctx, TM_BF16, oa.p, M, k, oa.ld * 2, 64, BK, &ta);
    else rc = get_tmap_2d(ctx, TM_BF16, oa.p, k, M, oa.ld * 2, BK, 128, &ta);
    if (rc) return rc;
    if ((rc = get_tmap_2d(ctx, TM_BF16, ob.p, N, k, ob.ld * 2, 64, BK, &tb))) return rc;
  }
  auto kern = gemm8_pair_kernel<KIND>;
  const void* key = reinterpret_cast<const void*>(kern);
  if (!ctx->smem_attr_done.count(key)) {
    GB_CUDA_CHECK(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES));
    ctx->smem_attr_done.insert(key);
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(GEMM8_THREADS, 1, 1);
  cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
  cfg.stream = ctx->stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto found = ctx->max_clusters.find(key);
  if (found == ctx->max_clusters.end()) {
    int n = 0;
    cfg.gridDim = dim3(2 * (ctx->num_sms / 2), 1, 1);
    GB_CUDA_CHECK(ctx, cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
    if (n <= 0) return set_error(ctx, GRILLY_ERR_UNSUPPORTED, "8-bit rows: no CTA pair fits on this GPU");
    found = ctx->max_clusters.emplace(key, n).first;
  }
  const int pairs = found->second;
  const long long tiles_m = (M + Cfg::TILE - 1) / Cfg::TILE, tiles_n = (N + Cfg::TILE - 1) / Cfg::TILE;
  if (tiles_m * tiles_n > 0x3fffffffll) return set_error(ctx, GRILLY_ERR_UNSUPPORTED, "8-bit rows: too many tiles");
  g.M = M; g.N = N;
  g.tiles_m = static_cast<int>(tiles_m);
  g.tiles_n = static_cast<int>(tiles_n);
  g.tile_group = 8;
  g.k_blocks = static_cast<int>((k + BK - 1) / BK);
  g.err = ctx->err_dev;
  const int elt = g.out_bf16 ? 2 : 4;
  // parts along k until every pair has a tile
  const int tiles = g.tiles_m * g.tiles_n;
  const int want = std::max(1, std::min(pairs / tiles, g.k_blocks / 4));
  g.k_per_split = (g.k_blocks + want - 1) / want;
  g.splits = (g.k_blocks + g.k_per_split - 1) / g.k_per_split;
  if (static_cast<long long>(tiles) * g.splits > 0x3fffffffll) return set_error(ctx, GRILLY_ERR_UNSUPPORTED, "8-bit rows: too many tiles");
  g.by_tiles = Divisor(tiles);
  g.by_group_tiles = Divisor(g.tile_group * g.tiles_n);
  g.by_group = Divisor(g.tile_group);
  g.by_last_group = Divisor(std::max(1, g.tiles_m % g.tile_group));
  const double bytes = (kInt8 ? 1.0 : 2.0) * (static_cast<double>(M) * k + static_cast<double>(N) * k) + static_cast<double>(M) * N * elt;
  const int pi = prof_begin(ctx, PROF_GEMM, 2.0 * M * static_cast<double>(N) * k, bytes);
  cfg.gridDim = dim3(2 * std::min(pairs, tiles * g.splits), 1, 1);
  CUtensorMap to = ta;
  g.wide_store = g.ld_out * elt % 16 == 0 && reinterpret_cast<uintptr_t>(g.out) % 16 == 0;
  if (g.splits == 1) {
    // 64 bytes of 32 rows per store, cut off at the edges
    if (g.wide_store && (rc = get_tmap_2d(ctx, g.out_bf16 ? TM_BF16 : TM_F32, g.out, N, M, g.ld_out * elt, 64 / elt, 32, &to, TM_SW64))) return rc;
    GB_CUDA_CHECK(ctx, cudaLaunchKernelEx(&cfg, kern, ta, tb, to, g));
    ctx->launches++;
  } else {
    // planes of whole tiles, so that a store at the lower edge of one does not reach into the next
    Rows8Scratch ws(ctx);
    const long long ld_ws = (N + 3) / 4 * 4ll, plane_rows = tiles_m * Cfg::TILE;
    if ((rc = ws.take(static_cast<size_t>(g.splits) * plane_rows * ld_ws * 4))) return rc;
    Gemm8Args part = g;
    part.out = ws.p;
    part.ld_out = ld_ws;
    part.raw = part.wide_store = 1;
    if ((rc = get_tmap_2d(ctx, TM_F32, ws.p, N, g.splits * plane_rows, ld_ws * 4, 16, 32, &to, TM_SW64))) return rc;
    GB_CUDA_CHECK(ctx, cudaLaunchKernelEx(&cfg, kern, ta, tb, to, part));
    const long long pieces = M * ((N + 3) / 4);
    gemm8_join_kernel<KIND><<<static_cast<unsigned>(std::min<long long>((pieces + 255) / 256, ctx->num_sms * 8ll)), 256, 0, ctx->stream>>>(
        g, static_cast<const uint32_t*>(ws.p), ld_ws, plane_rows * ld_ws);
    ctx->launches += 2;
    GB_CUDA_CHECK(ctx, cudaGetLastError());
  }
  prof_end(ctx, pi);
  return GRILLY_OK;
}

template <int NT>
void launch_few(grilly_ctx* ctx, const FewArgs& a) {
  linear_q8_few_kernel<NT><<<(a.N + 15) / 16, 256, 0, ctx->stream>>>(a);
}

// bf16 rows that TMA can read: the tensor itself, or a copy with padded rows in `scratch`
int tma_rows(grilly_ctx* ctx, const void* x, long long rows, int n, Rows8Scratch& scratch, Operand* out) {
  if (n % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0) {
    *out = {x, n};
    return GRILLY_OK;
  }
  const int ld = (n + 7) / 8 * 8;
  if (int rc = scratch.take(static_cast<size_t>(rows) * ld * 2)) return rc;
  pitch_rows_kernel<<<static_cast<unsigned>(std::min<long long>((rows + 7) / 8, ctx->num_sms * 16ll)), 256, 0, ctx->stream>>>(
      static_cast<const __nv_bfloat16*>(x), static_cast<__nv_bfloat16*>(scratch.p), rows, n, ld);
  ctx->launches++;
  GB_CUDA_CHECK(ctx, cudaGetLastError());
  *out = {scratch.p, ld};
  return GRILLY_OK;
}

int column_sums(grilly_ctx* ctx, const __nv_bfloat16* g, float* out, long long M, int N) {
  const bool wide = N % 8 == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0;
  const int across = wide ? (N / 8 + 255) / 256 : (N + 255) / 256;
  const int blocks = static_cast<int>(std::max<long long>(1, std::min<long long>((M + 31) / 32, ctx->num_sms * 6ll / across)));
  const long long per = (M + blocks - 1) / blocks;
  Rows8Scratch ws(ctx);
  if (int rc = ws.take(sizeof(float) * static_cast<size_t>(blocks) * N)) return rc;
  float* partial = static_cast<float*>(ws.p);
  if (wide) column_sums_kernel<8><<<dim3(across, blocks), 256, 0, ctx->stream>>>(g, partial, M, N, per);
  else column_sums_kernel<1><<<dim3(across, blocks), 256, 0, ctx->stream>>>(g, partial, M, N, per);
  sum_partials_kernel<<<(N + 31) / 32, 512, 0, ctx->stream>>>(partial, out, blocks, N);
  ctx->launches += 2;
  GB_CUDA_CHECK(ctx, cudaGetLastError());
  return GRILLY_OK;
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
    const int out_bf16 = (flags & GRILLY_FLAG_OUT_BF16) ? 1 : 0;
    if (M <= FEW_TOKENS) {
      const FewArgs a{static_cast<const int8_t*>(xq), xs, static_cast<const int8_t*>(wq), ws, bias, y, static_cast<int>(M), N, K, ldx, ldw, act, out_bf16};
      const int pi = prof_begin(ctx, PROF_GEMM, 2.0 * M * N * K, static_cast<double>(N) * K + M * (K + (out_bf16 ? 2.0 : 4.0) * N));
      if (M <= 8) launch_few<1>(ctx, a);
      else if (M <= 16) launch_few<2>(ctx, a);
      else launch_few<4>(ctx, a);
      prof_end(ctx, pi);
      ctx->launches++;
      GB_CUDA_CHECK(ctx, cudaGetLastError());
      return GRILLY_OK;
    }
    Gemm8Args g{};
    g.out = y; g.ld_out = N; g.out_bf16 = out_bf16;
    g.row_scale = xs; g.col_scale = ws; g.bias = bias; g.act = act;
    return launch_gemm8<Gemm8Kind::Q8>(ctx, {xq, ldx}, {wq, ldw}, M, N, K, g);
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
    if (M == 0) {
      if (gw) GB_CUDA_CHECK(ctx, cudaMemsetAsync(gw, 0, static_cast<size_t>(N) * K * (bf16 ? 2 : 4), ctx->stream));
      if (gbias) GB_CUDA_CHECK(ctx, cudaMemsetAsync(gbias, 0, sizeof(float) * N, ctx->stream));
      return GRILLY_OK;
    }
    int rc;
    Operand g{}, weights{};
    Rows8Scratch g_rows(ctx), w_rows(ctx), x_rows(ctx);
    if ((gx || gw) && (rc = tma_rows(ctx, go, M, N, g_rows, &g))) return rc;
    if (gx) {
      if ((rc = tma_rows(ctx, w, N, K, w_rows, &weights))) return rc;
      Gemm8Args a{};
      a.out = gx; a.ld_out = K; a.out_bf16 = bf16;
      if ((rc = launch_gemm8<Gemm8Kind::DGRAD>(ctx, g, weights, M, K, N, a))) return rc;
    }
    if (gw) {
      if ((rc = x_rows.take(static_cast<size_t>(M) * ldx * 2))) return rc;
      const long long pieces = M * (ldx / 16);
      expand_rows_kernel<<<static_cast<unsigned>(std::min<long long>((pieces + 255) / 256, ctx->num_sms * 32ll)), 256, 0, ctx->stream>>>(
          static_cast<const int8_t*>(xq), xs, static_cast<__nv_bfloat16*>(x_rows.p), pieces, static_cast<int>(ldx / 16));
      ctx->launches++;
      Gemm8Args a{};
      a.out = gw; a.ld_out = K; a.out_bf16 = bf16;
      if ((rc = launch_gemm8<Gemm8Kind::WGRAD>(ctx, g, {x_rows.p, ldx}, N, K, M, a))) return rc;
    }
    if (gbias && (rc = column_sums(ctx, static_cast<const __nv_bfloat16*>(go), gbias, M, N))) return rc;
    return GRILLY_OK;
  });
}

}  // extern "C"
