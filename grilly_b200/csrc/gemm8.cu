// Matrix products over 8-bit rows: y = act(s_x s_w x_q W_q^T + b), and the backward pass of a linear layer whose saved
// input is in 8-bit rows. The definitions stand with the entry points in include/grilly_b200.h.
#include "rows8.h"
#include "rows8_sum.cuh"
#include "gemm8.cuh"
#include <algorithm>
#include <initializer_list>

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

// 16 features per block; its warps walk K in pieces of 64. Both operands come straight from memory in 16-byte pieces: the
// sum over k does not care which k a lane calls its own, so lane t of four takes 16 consecutive bytes of a row and feeds
// them to two MMAs as if they were the fragment's columns, the same for weights and tokens. Rows past the end repeat the
// last one (their results are dropped); bytes past K are zeroed on the tokens' side. The warps' sums join in shared memory.
// 16384 x 4096 weights: 15.8 us for one token, 17.2 us for 16 (4 TB/s with about 3 us of start and end in it).
template <int NT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) linear_q8_few_kernel(const FewArgs a) {
  __shared__ int red[WARPS][16][8 * NT];
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
  for (int k = warp * 64; k < a.K; k += WARPS * 64) {
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
  for (int o = threadIdx.x; o < 16 * 8 * NT; o += 32 * WARPS) {
    const int f = f0 + (o & 15), m = o >> 4;
    if (f >= a.N || m >= a.M) continue;
    int s = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += red[w][o & 15][m];
    const float v = gemm8_act(fmaf(static_cast<float>(s) * __ldg(a.xs + m), __ldg(a.ws + f), a.bias ? __ldg(a.bias + f) : 0.f), a.act);
    const long long at = static_cast<long long>(m) * a.N + f;
    if (a.out_bf16) static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16(v);
    else static_cast<float*>(a.y)[at] = v;
  }
}

// ---------------------------------------------------------------- operands of the backward pass
// q * scale rounded to bf16, rows of ld values (what lies past the features is never read as a column): piece i of 16 bytes
__device__ __forceinline__ void expand_piece(const uint4 w, float s, __nv_bfloat16* y, long long i) {
  const uint32_t in[4] = {w.x, w.y, w.z, w.w};
  const F2 s2(s, s), offset(-8388736.f, -8388736.f);
  uint32_t out[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // signed bytes as floats: byte + 128 below the bits of 2^23, then the offset taken off; exact
    const uint32_t u = in[j] ^ 0x80808080u;
    const F2 lo(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)));
    const F2 hi(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443)));
    out[2 * j] = mul2(add2(lo, offset), s2).bf16();
    out[2 * j + 1] = mul2(add2(hi, offset), s2).bf16();
  }
  uint4* yp = reinterpret_cast<uint4*>(y) + 2 * i;
  yp[0] = make_uint4(out[0], out[1], out[2], out[3]);
  yp[1] = make_uint4(out[4], out[5], out[6], out[7]);
}
// 16 bytes from a 16-byte boundary on, 0 for values outside the tensor [first, last)
__device__ __forceinline__ uint4 load16_inside(const uint8_t* p, const uint8_t* first, const uint8_t* last) {
  if (p >= first && p + 16 <= last) return __ldg(reinterpret_cast<const uint4*>(p));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (p + 2 * j >= first && p + 2 * j < last) w[j / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + 2 * j)) << (j % 2 * 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// 8 bf16 values wherever they start, those from `left` on as 0. INSIDE: the aligned vectors that hold them are.
template <bool INSIDE>
__device__ __forceinline__ uint4 load_8(const __nv_bfloat16* x, const uint8_t* first, const uint8_t* last, int left) {
  const uint8_t* p = reinterpret_cast<const uint8_t*>(x);
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
  uint4 a, b;
  if constexpr (INSIDE) {
    a = __ldg(reinterpret_cast<const uint4*>(p - off));
    b = __ldg(reinterpret_cast<const uint4*>(p - off) + (off ? 1 : 0));
  } else {
    a = load16_inside(p - off, first, last);
    b = 2 * left + off > 16 && off ? load16_inside(p - off + 16, first, last) : make_uint4(0, 0, 0, 0);
  }
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int k = 0; k < 6; ++k) w[k] = off & 8 ? w[k + 2] : w[k];
#pragma unroll
  for (int k = 0; k < 5; ++k) w[k] = off & 4 ? w[k + 1] : w[k];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], (off & 2) * 8);
  if (left < 8) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (left <= 2 * k) w[k] = 0;
      else if (left == 2 * k + 1) w[k] &= 0xffffu;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// A block's rows of g, 256 columns of them: their sums to partial[block][n] (or null), and the rows themselves to a copy
// whose rows are ld apart (or null). 32 threads across with 8 columns each, 8 threads per column over every 8th row, added
// in turn. ANY: rows start anywhere (the 8 rows of a step have their own distances from a boundary, every step the same).
template <bool ANY>
__device__ __forceinline__ void sum_columns(const __nv_bfloat16* g, float* partial, __nv_bfloat16* copy, int ld, long long M, int N, int across, int block,
                                            long long rows_per_block, float (&part)[8][256]) {
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int n = (across * 32 + tx) * 8;
  const long long r0 = block * rows_per_block, r1 = min(M, r0 + rows_per_block);
  const uint8_t *first = reinterpret_cast<const uint8_t*>(g), *last = reinterpret_cast<const uint8_t*>(g + M * N);
  F2 acc[4] = {F2(0.f, 0.f), F2(0.f, 0.f), F2(0.f, 0.f), F2(0.f, 0.f)};
  auto take = [&](long long r, uint4 t) {
    if (ANY && copy) *reinterpret_cast<uint4*>(copy + r * ld + n) = t;
    const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = add2(acc[j], F2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u)));
  };
  if (n < N) {
    long long r = r0 + ty;
    if constexpr (ANY) {
      // rows 28 bytes away from both ends of the tensor go without checks: a row's last vector ends at most that far behind it
      const long long edge = (13 + N) / N, to = min(r1, M - edge);
      for (; r < r1 && r < edge; r += 8) take(r, load_8<false>(g + r * N + n, first, last, N - n));
#pragma unroll 8
      for (; r < to; r += 8) take(r, load_8<true>(g + r * N + n, first, last, N - n));
      for (; r < r1; r += 8) take(r, load_8<false>(g + r * N + n, first, last, N - n));
    } else {
#pragma unroll 8
      for (; r < r1; r += 8) take(r, __ldg(reinterpret_cast<const uint4*>(g + r * N + n)));
    }
  }
  if (!partial) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j].get(part[ty][(2 * j) * 32 + tx], part[ty][(2 * j + 1) * 32 + tx]);
  __syncthreads();
  const int c = threadIdx.x;               // column c of the block's 256: thread c / 8's value c % 8
  if (across * 256 + c < N) {
    const int at = (c % 8) * 32 + c / 8;
    float sum = part[0][at];
#pragma unroll
    for (int i = 1; i < 8; ++i) sum += part[i][at];
    partial[static_cast<long long>(block) * N + across * 256 + c] = sum;
  }
}
// What the tensor-core launch reads, and the column sums beside it (16384 x 4096, 4096 columns: 335 MB in 60 us): the first
// sum_blocks * across blocks sum columns of grad_out and, where TMA cannot read its rows, copy them; the next w_blocks copy
// such weights (COPIES), the others expand the 8-bit rows.
struct PrepareArgs {
  const int8_t* q;
  const float* scale;
  __nv_bfloat16* x;
  long long pieces;
  Divisor per_row;
  const __nv_bfloat16* g;
  float* partial;
  __nv_bfloat16* g_copy;
  long long M, rows_per_block;
  int N, ld_g, across, sum_blocks;
  const __nv_bfloat16* w;
  __nv_bfloat16* w_copy;
  int K, ld_w, w_blocks;
};
template <bool COPIES>
__global__ void __launch_bounds__(256) prepare_kernel(const __grid_constant__ PrepareArgs a) {
  __shared__ float part[8][256];
  const unsigned sums = a.sum_blocks * a.across;
  if (blockIdx.x < sums) {
    const int block = blockIdx.x / a.across, across = blockIdx.x - block * a.across;
    sum_columns<COPIES>(a.g, a.partial, a.g_copy, a.ld_g, a.M, a.N, across, block, a.rows_per_block, part);
    return;
  }
  if (COPIES && blockIdx.x < sums + a.w_blocks) {   // a warp per row
    const uint8_t *first = reinterpret_cast<const uint8_t*>(a.w), *last = reinterpret_cast<const uint8_t*>(a.w + static_cast<long long>(a.N) * a.K);
    for (long long row = (blockIdx.x - sums) * 8ll + (threadIdx.x >> 5); row < a.N; row += a.w_blocks * 8ll) {
#pragma unroll 4
      for (int k = (threadIdx.x & 31) * 8; k < a.K; k += 256)
        *reinterpret_cast<uint4*>(a.w_copy + row * a.ld_w + k) = load_8<false>(a.w + row * a.K + k, first, last, a.K - k);
    }
    return;
  }
  // 4 pieces per thread and turn, their loads together
  const unsigned before = sums + (COPIES ? a.w_blocks : 0);
  const long long step = (gridDim.x - before) * 1024ll;
  for (long long base = (blockIdx.x - before) * 1024ll + threadIdx.x; base < a.pieces; base += step) {
    uint4 w[4];
    float scale[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long i = min(base + u * 256, a.pieces - 1);
      w[u] = __ldg(reinterpret_cast<const uint4*>(a.q) + i);
      scale[u] = __ldg(a.scale + (a.pieces < (1ll << 31) ? a.per_row.quotient(static_cast<int>(i)) : i / a.per_row.d));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (base + u * 256 < a.pieces) expand_piece(w[u], scale[u], a.x, base + u * 256);
  }
}
// ---------------------------------------------------------------- launches
struct Operand {
  const void* p;
  long long ld;      // elements between rows
};

// Geometry of C [M][N] over k, in parts along k where its tiles are fewer than the CTA pairs.
int plan_gemm8(grilly_ctx* ctx, Gemm8Args& g, long long M, int N, long long k, int bk, int pairs) {
  constexpr int TILE = Gemm8Cfg<true>::TILE;
  if (M > 0x7fffff00ll || k > 0x7fffff00ll || N > 0x7fffff00) return set_error(ctx, GRILLY_ERR_UNSUPPORTED, "8-bit rows: more than 2^31 - 256 rows");
  g.M = M; g.N = N;
  const long long tiles_m = (M + TILE - 1) / TILE, tiles_n = (N + TILE - 1) / TILE;
  g.k_blocks = static_cast<int>((k + bk - 1) / bk);
  const long long tiles = tiles_m * tiles_n;
  // parts of at least 16 k-blocks, and none of a product under 48: the join's launch and its workspace cost about as much as
  // 16 k-blocks (256 x 4096 x 4096, 32 k-blocks: 14 us in one launch, 10 + 5 us in four parts)
  const int want = g.k_blocks < 48 ? 1 : static_cast<int>(std::max(1ll, std::min<long long>(pairs / tiles, g.k_blocks / 16)));
  g.k_per_split = (g.k_blocks + want - 1) / want;
  g.splits = (g.k_blocks + g.k_per_split - 1) / g.k_per_split;
  if (tiles * g.splits > 0x1fffffffll) return set_error(ctx, GRILLY_ERR_UNSUPPORTED, "8-bit rows: too many tiles");
  g.tiles_m = static_cast<int>(tiles_m);
  g.tiles_n = static_cast<int>(tiles_n);
  g.tile_group = 8;
  g.by_tiles = Divisor(static_cast<uint32_t>(tiles));
  g.by_group_tiles = Divisor(g.tile_group * g.tiles_n);
  g.by_group = Divisor(g.tile_group);
  g.by_last_group = Divisor(std::max(1, g.tiles_m % g.tile_group));
  const int elt = g.out_bf16 ? 2 : 4;
  g.wide_store = g.ld_out * elt % 16 == 0 && reinterpret_cast<uintptr_t>(g.out) % 16 == 0;
  return GRILLY_OK;
}

// A split product's parts: planes of whole tiles, so that a store at the lower edge of one does not reach into the next.
long long part_ld(const Gemm8Args& g) { return (g.N + 3) / 4 * 4ll; }
long long part_rows(const Gemm8Args& g) { return static_cast<long long>(g.tiles_m) * Gemm8Cfg<true>::TILE; }
size_t part_bytes(const Gemm8Args& g) { return g.splits > 1 ? static_cast<size_t>(g.splits) * part_rows(g) * part_ld(g) * 4 : 0; }

// Tensor maps of one product, and where its parts go (`parts`: part_bytes) when it is split.
int map_gemm8(grilly_ctx* ctx, bool int8, Operand oa, Operand ob, long long k, Gemm8Args& g, Gemm8Maps& m, uint32_t* parts, Gemm8Finish& f, int which) {
  int rc;
  if (int8) {
    if ((rc = get_tmap_2d(ctx, TM_U8, oa.p, k, g.M, oa.ld, 128, 128, &m.a))) return rc;
    if ((rc = get_tmap_2d(ctx, TM_U8, ob.p, k, g.N, ob.ld, 128, 128, &m.b))) return rc;
  } else {
    if (g.a_across) rc = get_tmap_2d(ctx, TM_BF16, oa.p, g.M, k, oa.ld * 2, 64, 64, &m.a);
    else rc = get_tmap_2d(ctx, TM_BF16, oa.p, k, g.M, oa.ld * 2, 64, 128, &m.a);
    if (rc) return rc;
    if ((rc = get_tmap_2d(ctx, TM_BF16, ob.p, g.N, k, ob.ld * 2, 64, 64, &m.b))) return rc;
  }
  m.out = m.a;
  const int elt = g.out_bf16 ? 2 : 4;
  f.pieces[which] = 0;
  if (g.splits == 1) {
    // 64 bytes of 32 rows per store, cut off at the edges
    return g.wide_store ? get_tmap_2d(ctx, g.out_bf16 ? TM_BF16 : TM_F32, g.out, g.N, g.M, g.ld_out * elt, 64 / elt, 32, &m.out, TM_SW64) : GRILLY_OK;
  }
  f.job[which] = g;
  f.ws[which] = parts;
  f.ld_ws[which] = part_ld(g);
  f.plane[which] = part_rows(g) * part_ld(g);
  f.pieces[which] = g.M * (part_ld(g) / 4);
  f.per_row[which] = Divisor(static_cast<uint32_t>(part_ld(g) / 4));
  g.out = parts;
  g.ld_out = part_ld(g);
  g.raw = g.wide_store = 1;
  return get_tmap_2d(ctx, TM_F32, parts, g.N, g.splits * part_rows(g), g.ld_out * 4, 16, 32, &m.out, TM_SW64);
}

template <bool kInt8>
int pairs_that_fit(grilly_ctx* ctx, cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, int* pairs) {
  auto kern = gemm8_pair_kernel<kInt8>;
  const void* key = reinterpret_cast<const void*>(kern);
  if (!ctx->smem_attr_done.count(key)) {
    GB_CUDA_CHECK(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Gemm8Cfg<kInt8>::SMEM_BYTES));
    ctx->smem_attr_done.insert(key);
  }
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = 2;
  attr->val.clusterDim.y = 1;
  attr->val.clusterDim.z = 1;
  cfg.blockDim = dim3(GEMM8_THREADS, 1, 1);
  cfg.dynamicSmemBytes = Gemm8Cfg<kInt8>::SMEM_BYTES;
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
  *pairs = found->second;
  return GRILLY_OK;
}

template <bool kInt8>
int launch_gemm8(grilly_ctx* ctx, cudaLaunchConfig_t& cfg, int pairs, const Gemm8Maps* maps, Gemm8Jobs& jobs, bool follows) {
  int items = 0;
  double flops = 0, bytes = 0;
  for (int j = 0; j < jobs.count; ++j) {
    const Gemm8Args& g = jobs.job[j];
    jobs.items[j] = g.tiles_m * g.tiles_n * g.splits;
    items += jobs.items[j];
    const double k = static_cast<double>(g.k_blocks) * (kInt8 ? 128 : 64);
    flops += 2.0 * g.M * g.N * k;
    bytes += (kInt8 ? 1.0 : 2.0) * (static_cast<double>(g.M) + g.N) * k + static_cast<double>(g.M) * g.N * (g.out_bf16 ? 2 : 4);
  }
  const int P = std::min(pairs, items);
  jobs.ahead_from = jobs.items[0] % P;
  jobs.ahead = 0;
  if (jobs.count > 1 && jobs.ahead_from) {
    const int late = P - jobs.ahead_from;
    jobs.ahead = std::min(jobs.job[0].k_per_split / jobs.job[1].k_per_split, jobs.items[1] / late);
  }
  jobs.err = ctx->err_dev;
  cfg.gridDim = dim3(2 * P, 1, 1);
  if (follows) cfg.attrs[cfg.numAttrs++] = early_launch();
  const int pi = prof_begin(ctx, PROF_GEMM, flops, bytes);
  GB_CUDA_CHECK(ctx, cudaLaunchKernelEx(&cfg, gemm8_pair_kernel<kInt8>, maps[0], maps[jobs.count - 1], jobs));
  prof_end(ctx, pi);
  ctx->launches++;
  return GRILLY_OK;
}

// The second launch: parts joined, column sums totalled; nothing where neither is there.
template <bool kInt8>
int launch_finish(grilly_ctx* ctx, Gemm8Finish& f) {
  const long long pieces = std::max(f.pieces[0], f.pieces[1]);
  f.sum_at = static_cast<unsigned>(std::min<long long>((pieces + 511) / 512, ctx->num_sms * 4ll));
  const unsigned grid = f.sum_at + (f.sums ? (f.F + 31) / 32 : 0);
  if (!grid) return GRILLY_OK;
  GB_CUDA_CHECK(ctx, launch_following(ctx->stream, gemm8_finish_kernel<kInt8>, grid, 512, f));
  ctx->launches++;
  return GRILLY_OK;
}

// Which products go to linear_q8_few_kernel, which to the tensor-core tiles; the results are the same. Up to 16 tokens cost
// about as much as one, the weights' bytes (us here | tiles at 16 tokens: 1536 x 384 2.3 | 6.1, 4096 x 4096 7.0 | 15.2,
// 16384 x 4096 17.2 | 20.3, 65536 x 512 13.7 | 14.2, 100000 x 768 24.0 | 24.5), but where few blocks share a long row, which
// tiles split along k (1024 x 16384 14.1 | 14.1, 2048 x 32768 28.1 | 21.8, 512 x 65536 48.9 | 18.3, 4096 x 32768 33.2 | 35.7).
// With more tokens their bytes, read again for every 16 features, and the mma.sync pipe count. At 32 tokens: 4096 x 4096
// 10.9 | 15.2, 6144 x 4096 12.9 | 15.6, 6144 x 384 6.5 | 6.9, 8192 x 384 8.3 | 6.9, 8192 x 4096 19.9 | 16.1, 2048 x 8192
// 15.2 | 13.7, 16384 x 4096 21.9 | 19.0, 4096 x 16384 30.4 | 21.5.
bool few_tokens(long long M, int N, int K) {
  if (M <= 16) return K <= 16384 || N > 2048;
  return M <= 32 && N <= 6144 && K <= 4096;
}

template <int NT>
void launch_few(grilly_ctx* ctx, const FewArgs& a) {
  // about 4096 warps on the GPU, whatever N: many blocks of 4 warps, or few of 16 that share a longer row (for a single
  // token 4096 x 4096 takes 6.7, 4.2 and 3.9 us with 4, 8 and 16 warps, 16384 x 4096 15.7, 16.6 and 18.6 us). 32 tokens
  // make the warps' join dearer: 8 (4096 x 4096 takes 14.8, 10.9 and 14.5 us, 6144 x 1024 6.7, 7.7 and 13.5).
  const unsigned blocks = (a.N + 15) / 16;
  if constexpr (NT == 4) {
    linear_q8_few_kernel<NT, 8><<<blocks, 256, 0, ctx->stream>>>(a);
  } else {
    if (blocks > 512) linear_q8_few_kernel<NT, 4><<<blocks, 128, 0, ctx->stream>>>(a);
    else if (blocks > 256) linear_q8_few_kernel<NT, 8><<<blocks, 256, 0, ctx->stream>>>(a);
    else linear_q8_few_kernel<NT, 16><<<blocks, 512, 0, ctx->stream>>>(a);
  }
}

// bf16 rows that TMA can read as they are; others are copied to rows of a multiple of 8 values
bool tma_reads(const void* x, int n) { return n % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0; }
int pitch_of(int n) { return (n + 7) / 8 * 8; }
size_t pitch_bytes(const void* x, long long rows, int n) { return tma_reads(x, n) ? 0 : static_cast<size_t>(rows) * pitch_of(n) * 2; }

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
    if (N > ROWS8_MAX_FEATURES) return set_error(ctx, GRILLY_ERR_UNSUPPORTED, "linear_q8: more than 2^30 output features");
    if (K > 131071) return set_error(ctx, GRILLY_ERR_UNSUPPORTED, "linear_q8: more than 131071 features can overflow the 32-bit sums");
    if (act < GRILLY_ACT_NONE || act > GRILLY_ACT_RELU) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "linear_q8: unknown activation");
    if (M == 0) return GRILLY_OK;
    if (!y) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "linear_q8: null output");
    const int out_bf16 = (flags & GRILLY_FLAG_OUT_BF16) ? 1 : 0;
    const Rows8Span outs[] = {{y, M * N * (out_bf16 ? 2 : 4), 0, out_bf16 ? 2 : 4}};
    const Rows8Span ins[] = {{xq, M * ldx}, {xs, 4 * M}, {wq, N * ldw}, {ws, 4ll * N}, {bias, 4ll * N}};
    if (int rc = rows8_memory(ctx, "linear_q8", outs, ins)) return rc;
    if (few_tokens(M, N, K)) {
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
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    int pairs = 0, rc;
    if ((rc = pairs_that_fit<true>(ctx, cfg, attr, &pairs))) return rc;
    Gemm8Jobs jobs{};
    Gemm8Maps maps;
    Gemm8Finish finish{};
    Rows8Scratch parts(ctx);
    jobs.count = 1;
    Gemm8Args& g = jobs.job[0];
    g.out = y; g.ld_out = N; g.out_bf16 = out_bf16;
    g.row_scale = xs; g.col_scale = ws; g.bias = bias; g.act = act;
    if ((rc = plan_gemm8(ctx, g, M, N, K, 128, pairs))) return rc;
    const size_t at = parts.reserve(part_bytes(g));
    if ((rc = parts.take())) return rc;
    if ((rc = map_gemm8(ctx, true, {xq, ldx}, {wq, ldw}, K, g, maps, parts.at<uint32_t>(at), finish, 0))) return rc;
    if ((rc = launch_gemm8<true>(ctx, cfg, pairs, &maps, jobs, false))) return rc;
    return launch_finish<true>(ctx, finish);
  });
}

int grilly_linear_backward_q8(grilly_ctx* ctx, const void* go, const void* xq, const float* xs, const void* w, void* gx, void* gw, float* gbias,
                              long long M, int N, int K, long long ldx, int flags) {
  return rows8_entry(ctx, [&]() -> int {
    if (int rc = rows8_check(ctx, "linear_backward_q8: x", xq, xs, M, K, ldx)) return rc;
    if (N < 1) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "linear_backward_q8: N must be positive");
    if (N > ROWS8_MAX_FEATURES) return set_error(ctx, GRILLY_ERR_UNSUPPORTED, "linear_backward_q8: more than 2^30 output features");
    const bool bf16 = flags & GRILLY_FLAG_OUT_BF16;
    if (M > 0 && !go) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "linear_backward_q8: null gradient");
    if (gx && !w) return set_error(ctx, GRILLY_ERR_INVALID_ARG, "linear_backward_q8: grad_x needs the weights");
    const int elt = bf16 ? 2 : 4;
    const Rows8Span outs[] = {{gx, M * K * elt, 0, elt}, {gw, static_cast<long long>(N) * K * elt, 0, elt}, {gbias, 4ll * N}};
    const Rows8Span ins[] = {{go, M * N * 2, 0, 2}, {xq, M * ldx}, {xs, 4 * M}, {w, static_cast<long long>(N) * K * 2, 0, 2}};
    if (int rc = rows8_memory(ctx, "linear_backward_q8", outs, ins)) return rc;
    if (M == 0) {
      if (gw) GB_CUDA_CHECK(ctx, cudaMemsetAsync(gw, 0, static_cast<size_t>(N) * K * (bf16 ? 2 : 4), ctx->stream));
      if (gbias) GB_CUDA_CHECK(ctx, cudaMemsetAsync(gbias, 0, sizeof(float) * N, ctx->stream));
      return GRILLY_OK;
    }
    int rc, pairs = 0;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    if ((rc = pairs_that_fit<false>(ctx, cfg, attr, &pairs))) return rc;
    // the products, the one with the longer sums first
    Gemm8Jobs jobs{};
    bool is_w[2] = {};
    const bool w_first = gw && (!gx || M >= N);
    for (int j = 0; j < 2; ++j) {
      const bool w_job = (j == 0) == w_first;
      if (w_job ? !gw : !gx) continue;
      is_w[jobs.count] = w_job;
      Gemm8Args& a = jobs.job[jobs.count++];
      a.out = w_job ? gw : gx;
      a.ld_out = K;
      a.out_bf16 = bf16;
      a.a_across = w_job;
      if ((rc = plan_gemm8(ctx, a, w_job ? N : M, K, w_job ? M : N, 64, pairs))) return rc;
    }
    PrepareArgs p{};
    p.per_row = Divisor(1);
    const bool copy_g = jobs.count && !tma_reads(go, N), copy_w = gx && !tma_reads(w, K);
    if (gbias || copy_g) {
      p.across = (N + 255) / 256;
      p.sum_blocks = static_cast<int>(std::max<long long>(1, std::min<long long>((M + 63) / 64, ctx->num_sms * 4ll / p.across)));
    }
    Rows8Scratch scratch(ctx);
    const size_t at_g = scratch.reserve(copy_g ? pitch_bytes(go, M, N) : 0), at_w = scratch.reserve(copy_w ? pitch_bytes(w, N, K) : 0);
    const size_t at_x = scratch.reserve(gw ? static_cast<size_t>(M) * ldx * 2 : 0), at_sums = scratch.reserve(gbias ? sizeof(float) * static_cast<size_t>(p.sum_blocks) * N : 0);
    const size_t at_parts[2] = {scratch.reserve(part_bytes(jobs.job[0])), scratch.reserve(part_bytes(jobs.job[1]))};
    if ((rc = scratch.take())) return rc;
    Gemm8Finish finish{};
    // the checkpoint as bf16 rows, the column sums of grad_out by blocks of rows, copies
    unsigned blocks = 0;
    p.N = N;
    if (gbias || copy_g) {
      p.g = static_cast<const __nv_bfloat16*>(go);
      p.M = M;
      p.rows_per_block = (M + p.sum_blocks - 1) / p.sum_blocks;
      blocks = p.across * p.sum_blocks;
      if (copy_g) p.g_copy = scratch.at<__nv_bfloat16>(at_g);
      p.ld_g = pitch_of(N);
    }
    if (copy_w) {
      p.w = static_cast<const __nv_bfloat16*>(w);
      p.w_copy = scratch.at<__nv_bfloat16>(at_w);
      p.K = K;
      p.ld_w = pitch_of(K);
      p.w_blocks = static_cast<int>(std::min<long long>((N + 7) / 8, ctx->num_sms * 4ll));
      blocks += p.w_blocks;
    }
    if (gbias) {
      p.partial = scratch.at<float>(at_sums);
      finish.partial = p.partial;
      finish.sums = gbias;
      finish.blocks = p.sum_blocks;
      finish.F = N;
    }
    if (gw) {
      p.q = static_cast<const int8_t*>(xq);
      p.scale = xs;
      p.x = scratch.at<__nv_bfloat16>(at_x);
      p.pieces = M * (ldx / 16);
      p.per_row = Divisor(static_cast<uint32_t>(ldx / 16));
      blocks += static_cast<unsigned>(std::min<long long>((p.pieces + 1023) / 1024, ctx->num_sms * 4ll));
    }
    if (blocks) {
      const int pi = prof_begin(ctx, PROF_OTHER, 0.0, (gw ? 3.0 * M * K : 0.0) + (gbias || copy_g ? 2.0 * M * N : 0.0) + (copy_g ? 2.0 * M * N : 0.0) + (copy_w ? 4.0 * N * K : 0.0));
      if (copy_w || !tma_reads(go, N)) prepare_kernel<true><<<blocks, 256, 0, ctx->stream>>>(p);
      else prepare_kernel<false><<<blocks, 256, 0, ctx->stream>>>(p);
      prof_end(ctx, pi);
      ctx->launches++;
      GB_CUDA_CHECK(ctx, cudaGetLastError());
    }
    if (jobs.count) {
      const Operand g = copy_g ? Operand{p.g_copy, p.ld_g} : Operand{go, N}, weights = copy_w ? Operand{p.w_copy, p.ld_w} : Operand{w, K};
      Gemm8Maps maps[2];
      for (int j = 0; j < jobs.count; ++j) {
        const Operand b = is_w[j] ? Operand{scratch.at<void>(at_x), ldx} : weights;
        if ((rc = map_gemm8(ctx, false, g, b, is_w[j] ? M : N, jobs.job[j], maps[j], scratch.at<uint32_t>(at_parts[j]), finish, j))) return rc;
      }
      if ((rc = launch_gemm8<false>(ctx, cfg, pairs, maps, jobs, blocks > 0))) return rc;
    }
    return launch_finish<false>(ctx, finish);
  });
}

}  // extern "C"
