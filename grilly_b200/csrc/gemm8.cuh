// Matrix products of the 8-bit row operators on the tensor cores: C[M][N] = epilogue(sum over k of A(m, k) B(n, k)).
//
//   linear_q8            A = x_q [M][K], B = W_q [N][K], int8 along k (kind::i8, exact int32 sums)
//   linear_backward_q8   two products in one launch, bf16 with fp32 sums:
//     grad_x = grad_out W       A = grad_out [M][k] along k, B = W [k][N] across k
//     grad_W = grad_out^T x     A = grad_out [k][M], B = x [k][N], both across k
//
// A pair of CTAs shares one tcgen05.mma (cta_group::2): a 256 x 256 tile of C, of which each CTA loads 128 rows of A and
// 128 of B per k-block of 128 bytes and keeps 128 rows of the accumulator in its own tensor memory, twice, so that one
// tile is written while the next is computed. Roles per CTA: warp 0 TMA producer (own halves, bytes counted on the
// leader's barrier), warp 1 MMA issuer (leader) and TMEM allocation, 16 epilogue warps, and one warp that works out the next
// tile's place and brings its scales and bias into shared memory (left to the epilogue warps, 16 of them did the same
// integer work for 1000 of the 5000 cycles of a 384-deep tile, and waited for L2 twice).
// Every wait is bounded and reports through the device status word. Nothing is broadcast by TMA.
//
// A k-block costs 0.38 us whatever its type: 64 KB into the pair's shared memory, 512 cycles of MMA. 8192 x 8192 x 8192 int8
// takes 335 us (3280 TOP/s; 390 us once the power cap holds), both products of a backward pass at 16384 x 4096 x 4096 710 us
// (1550 TFLOP/s; 820 us under the cap). Where k is short the epilogue sets the pace: 32768 x 384 x 1536 with GELU 44 us,
// without 33 us, 18 us of it the main loop.
//
// Few tiles of a long product are split along k: every part stores its raw 32-bit sums to its own plane of a workspace and
// a second kernel adds the planes in order (no atomics: results repeat bit for bit).
#pragma once
#include "ptx.cuh"
#include "f32x2.cuh"
#include "rows8_sum.cuh"
#include "../../include/grilly_b200.h"
#include <cuda_bf16.h>

namespace gb {

// Division of 0 <= n < 2^31 by a number the host knows: n * m >> s with s = 31 + ceil(log2 d), m = floor(2^s / d) + 1. The
// error of m is at most 2^-31 of a quotient step for every such n, so the quotient is exact (Granlund and Montgomery).
struct Divisor {
  uint32_t d, m, s;
  Divisor() = default;
  __host__ explicit Divisor(uint32_t n) : d(n), s(31) {
    while ((1ull << (s - 31)) < n) ++s;
    m = static_cast<uint32_t>((1ull << s) / n + 1);
  }
  __device__ __forceinline__ int quotient(int n) const { return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * m) >> s); }
};

// One product of a launch.
struct Gemm8Args {
  long long M;
  int N;
  int a_across;               // bf16: A lies across k
  int tiles_m, tiles_n, tile_group, k_blocks;
  int splits, k_per_split;    // k-blocks per part
  Divisor by_tiles, by_group_tiles, by_group, by_last_group;   // tiles, group * tiles_n, group, tiles_m % group (or 1)
  // epilogue
  void* out;                  // C [M][N] fp32 or bf16, or the workspace [splits][M][ld_out] of raw sums
  long long ld_out;
  int out_bf16, raw;
  int wide_store;             // rows of C lie on 16-byte boundaries: TMA stores them
  const float* row_scale;     // Q8: per row and per column, and the bias
  const float* col_scale;
  const float* bias;
  int act;
};
struct Gemm8Maps {
  CUtensorMap a, b, out;
};
// The products of a launch and how the pairs share them: pair p of P takes the items (tile and part of k) p, p + P, ... of
// the first, then items of the second. Where the first does not divide evenly, the pairs from ahead_from on are one item
// short and take `ahead` items more of the second (the first's items are the longer ones).
struct Gemm8Jobs {
  Gemm8Args job[2];
  int count, items[2];
  int ahead_from, ahead;
  int* err;
};
struct Gemm8Walk {
  int p, P, first, j;
  __device__ Gemm8Walk(int pair, int pairs) : p(pair), P(pairs), first(pair), j(0) {}
  __device__ __forceinline__ bool next(const Gemm8Jobs& jobs, int& job, int& item) {
    if (first < jobs.items[0]) {
      job = 0;
      item = first;
      first += P;
      return true;
    }
    if (jobs.count < 2) return false;
    const int late = P - jobs.ahead_from, before = jobs.ahead * late;
    job = 1;
    if (p >= jobs.ahead_from) item = j < jobs.ahead ? j * late + p - jobs.ahead_from : before + (j - jobs.ahead) * P + p;
    else item = before + j * P + p;
    ++j;
    return item < jobs.items[1];
  }
};

// Where the epilogue finds its tile, double-buffered in shared memory.
struct Gemm8Place {
  long long row0;        // first row of the CTA's half
  int out_row;           // the same as a coordinate of the output's tensor map
  int col0, chunks;      // first column; blocks of 32 columns that lie in C
  int job;
};
static_assert(sizeof(Gemm8Place) <= 32, "Gemm8Place");
constexpr int GEMM8_EPI_WARPS = 16;
constexpr int GEMM8_PARAM_WARP = 2 + GEMM8_EPI_WARPS;
constexpr int GEMM8_THREADS = 32 * (GEMM8_PARAM_WARP + 1);

template <bool kInt8>
struct Gemm8Cfg {
  static constexpr int TILE = 256;
  static constexpr int HALF_BYTES = 128 * 128;               // 128 rows (or columns) x 128 bytes
  static constexpr int STAGE_BYTES = 2 * HALF_BYTES;
  static constexpr int STAGES = kInt8 ? 5 : 6;               // what fits beside the rest
  static constexpr int EPI_BYTES = 32 * 64;                  // per epilogue warp: 32 rows x 64 bytes of C on their way out
  static constexpr int PARAM_BYTES = 32 + (kInt8 ? (2 * TILE + 128) * 4 : 0);   // a Gemm8Place; column scales, bias, row scales
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + GEMM8_EPI_WARPS * EPI_BYTES + 2 * PARAM_BYTES + 1024 /*align slack*/ + 256 /*barriers*/;
  static constexpr int TMEM_COLS = 512;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory of one CTA");
};

// ---- epilogue arithmetic, two neighbouring columns at a time
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// v * sigmoid(z) with z = v for SiLU and z = 2 sqrt(2/pi) (v + 0.044715 v^3) for GELU (its tanh form: 0.5 v (1 + tanh(z / 2))).
// One exponential and one reciprocal, each within 2 ulp, keep the relative accuracy far below zero too, where 1 + tanh
// would cancel. Where 2^(-z log2 e) overflows, the reciprocal is 0 and so is the result.
template <int ACT>
__device__ __forceinline__ F2 gemm8_act2(F2 v) {
  constexpr float L2E = 1.4426950408889634f, S = 2.f * 0.7978845608028654f;
  if constexpr (ACT == GRILLY_ACT_RELU) {
    float a, b;
    v.get(a, b);
    return F2(a < 0.f ? 0.f : a, b < 0.f ? 0.f : b);
  } else if constexpr (ACT == GRILLY_ACT_GELU || ACT == GRILLY_ACT_SILU) {
    F2 z;
    if constexpr (ACT == GRILLY_ACT_GELU) z = mul2(v, fma2(mul2(v, v), F2(-S * L2E * 0.044715f, -S * L2E * 0.044715f), F2(-S * L2E, -S * L2E)));
    else z = mul2(v, F2(-L2E, -L2E));
    float a, b;
    z.get(a, b);
    add2(F2(fast_exp2(a), fast_exp2(b)), F2(1.f, 1.f)).get(a, b);
    return mul2(v, F2(fast_rcp(a), fast_rcp(b)));
  } else {
    return v;
  }
}
__device__ __forceinline__ float gemm8_act(float v, int act) {
  float a, b;
  switch (act) {
    case GRILLY_ACT_GELU: gemm8_act2<GRILLY_ACT_GELU>(F2(v, v)).get(a, b); return a;
    case GRILLY_ACT_SILU: gemm8_act2<GRILLY_ACT_SILU>(F2(v, v)).get(a, b); return a;
    case GRILLY_ACT_RELU: return v < 0.f ? 0.f : v;
    default: return v;
  }
}

// Tile of the persistent loop: row blocks are walked in groups so that the tiles of one moment share rows of A and B.
__device__ __forceinline__ void gemm8_tile(const Gemm8Args& a, int tile, int& m, int& n) {
  const int g = a.by_group_tiles.quotient(tile), first = g * a.tile_group;
  const int r = tile - g * static_cast<int>(a.by_group_tiles.d);
  const bool whole = first + a.tile_group <= a.tiles_m;
  n = whole ? a.by_group.quotient(r) : a.by_last_group.quotient(r);
  m = first + r - n * static_cast<int>(whole ? a.by_group.d : a.by_last_group.d);
}

// The last column of tiles, where at most 128 of its columns lie in C: half as wide (a k-block then costs 0.27 instead of
// 0.38 us). Each CTA of the pair still brings half of the tile's columns.
__device__ __forceinline__ bool gemm8_narrow(const Gemm8Args& a, int tn) { return a.N - tn * 256 <= 128; }

// The epilogue works on 32 rows x 16 columns at a time: a lane has 16 neighbouring columns of its row, as raw sums.
// int8: times the row's scale, times the column's scale plus bias (shared memory, the same address in every lane), activation.
template <int ACT>
__device__ __forceinline__ void gemm8_finish(uint32_t (&r)[16], float rs, const float* cs, const float* bias) {
  const F2 rs2(rs, rs);
  ulonglong2 c[4], d[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    c[j] = reinterpret_cast<const ulonglong2*>(cs)[j];
    d[j] = reinterpret_cast<const ulonglong2*>(bias)[j];
  }
#pragma unroll
  for (int j = 0; j < 16; j += 2) {
    F2 c2, d2;
    c2.v = j & 2 ? c[j / 4].y : c[j / 4].x;
    d2.v = j & 2 ? d[j / 4].y : d[j / 4].x;
    const F2 v(static_cast<float>(static_cast<int>(r[j])), static_cast<float>(static_cast<int>(r[j + 1])));
    float a, b;
    gemm8_act2<ACT>(fma2(mul2(v, rs2), c2, d2)).get(a, b);
    r[j] = __float_as_uint(a);
    r[j + 1] = __float_as_uint(b);
  }
}
__device__ __forceinline__ void gemm8_finish(uint32_t (&r)[16], float rs, const float* cs, const float* bias, int act) {
  switch (act) {
    case GRILLY_ACT_GELU: return gemm8_finish<GRILLY_ACT_GELU>(r, rs, cs, bias);
    case GRILLY_ACT_SILU: return gemm8_finish<GRILLY_ACT_SILU>(r, rs, cs, bias);
    case GRILLY_ACT_RELU: return gemm8_finish<GRILLY_ACT_RELU>(r, rs, cs, bias);
    default: return gemm8_finish<GRILLY_ACT_NONE>(r, rs, cs, bias);
  }
}
// 4 words of a lane's row of 64 bytes, as piece p; pieces are exchanged as TMA's 64-byte swizzle does, so neither side has
// bank conflicts
__device__ __forceinline__ void gemm8_stage(uint8_t* stage, int lane, int p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  *reinterpret_cast<uint4*>(stage + lane * 64 + ((p ^ ((lane >> 1) & 3)) << 4)) = make_uint4(a, b, c, d);
}
// The 16 columns from `first` on go to the warp's 2 KB of shared memory, rows of 64 bytes: 16 columns of 32 bits, or a half
// (h) of 32 columns of bf16. A full row leaves by one TMA store, cut off at the edges of C; where C's rows are not on
// 16-byte boundaries the lanes store the 64 bytes of a row themselves (16 bf16 columns at a time, 32 bytes, took 52 us
// instead of 40 for 16384 x 385 x 1537).
__device__ __forceinline__ void gemm8_write(const Gemm8Args& a, const CUtensorMap* tmap_out, const uint32_t (&r)[16], uint8_t* stage, long long row0,
                                            int out_row, int first, int h, int lane) {
  const bool half = a.out_bf16 && !a.raw;
  if (!(half && h == 1)) {
    // the warp's last store has left the staging rows (it may have been of the launch's other product, stored otherwise)
    if (lane == 0) tma_store_wait_read<0>();
    __syncwarp();
  }
  if (half) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = F2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])).bf16();
    gemm8_stage(stage, lane, 2 * h, w[0], w[1], w[2], w[3]);
    gemm8_stage(stage, lane, 2 * h + 1, w[4], w[5], w[6], w[7]);
    if (h == 0) return;
    first -= 16;
  } else {
#pragma unroll
    for (int p = 0; p < 4; ++p) gemm8_stage(stage, lane, p, r[4 * p], r[4 * p + 1], r[4 * p + 2], r[4 * p + 3]);
    if (first >= a.N) return;                                // the block's second half lies past C
  }
  if (a.wide_store) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(tmap_out, stage, first, out_row);
      tma_store_commit();
    }
    return;
  }
  __syncwarp();
  const int rows = static_cast<int>(a.M - row0 < 32 ? a.M - row0 : 32);
  if (half) {
    if (first + lane < a.N) {
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + row0 * a.ld_out + first + lane;
#pragma unroll 8
      for (int q = 0; q < rows; ++q, out += a.ld_out)
        *out = *reinterpret_cast<const __nv_bfloat16*>(stage + q * 64 + (((lane >> 3) ^ ((q >> 1) & 3)) << 4) + (lane & 7) * 2);
    }
  } else {
    const int c = lane & 15;
    if (first + c < a.N) {
      float* out = static_cast<float*>(a.out) + (row0 + (lane >> 4)) * a.ld_out + first + c;
#pragma unroll 8
      for (int q = lane >> 4; q < rows; q += 2, out += 2 * a.ld_out)
        *out = *reinterpret_cast<const float*>(stage + q * 64 + (((c >> 2) ^ ((q >> 1) & 3)) << 4) + (c & 3) * 4);
    }
  }
}

// kind::i8 over a pair, signed operands, 32-bit integer sums
__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor of kind::i8: 32-bit integer accumulator (2), both operands signed (1) and along k.
__host__ __device__ constexpr uint32_t make_idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

template <bool kInt8>
__global__ void __launch_bounds__(GEMM8_THREADS, 1)
gemm8_pair_kernel(const __grid_constant__ Gemm8Maps maps0, const __grid_constant__ Gemm8Maps maps1, const __grid_constant__ Gemm8Jobs jobs) {
  using Cfg = Gemm8Cfg<kInt8>;
  constexpr int STAGES = Cfg::STAGES;
  constexpr int BK = kInt8 ? 128 : 64;                         // k per stage
  constexpr int KSTEPS = 4;                                    // instructions per stage, 32 bytes of k each
  constexpr uint32_t ACROSS_STEP = 16 * 128;                   // bytes of an operand across k per instruction

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + STAGES * Cfg::STAGE_BYTES;
  uint8_t* params = epi + GEMM8_EPI_WARPS * Cfg::EPI_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(params + 2 * Cfg::PARAM_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tmem_full = empty_bar + STAGES;
  uint64_t* tmem_empty = tmem_full + 2;
  uint64_t* param_full = tmem_empty + 2;
  uint64_t* param_empty = param_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(param_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();                     // 0 = leader
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);                              // used in the leader only
      mbar_init(&empty_bar[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tmem_full[i], 1);
      mbar_init(&tmem_empty[i], 2 * GEMM8_EPI_WARPS);          // used in the leader only
      mbar_init(&param_full[i], 1);
      mbar_init(&param_empty[i], GEMM8_EPI_WARPS);
    }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&maps0.a);
    prefetch_tmap(&maps0.b);
    prefetch_tmap(&maps0.out);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_holder, Cfg::TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();                                              // the peer's barriers exist before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  wait_for_previous_kernel();                                  // what it writes is read from here on

  // a failed wait stops both CTAs: the peer's waits poll its own flag
  auto fail = [&](int code) {
    if (!*abort_flag) atomicCAS(jobs.err, 0, code);
    *abort_flag = 1;
    st_cluster_u32(map_to_cta(const_cast<int*>(abort_flag), rank ^ 1u), 1u);
  };
  // tile and k-blocks of an item
  auto place = [&](const Gemm8Args& a, int item, int& tm, int& tn, int& k0, int& k1) {
    const int part = a.by_tiles.quotient(item);
    gemm8_tile(a, item - part * static_cast<int>(a.by_tiles.d), tm, tn);
    k0 = part * a.k_per_split;
    k1 = min(a.k_blocks, k0 + a.k_per_split);
    return part;
  };
  Gemm8Walk walk(pair, num_pairs);
  int job, item;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs, own halves)
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      while (ok && walk.next(jobs, job, item)) {
        const Gemm8Args& a = jobs.job[kInt8 ? 0 : job];
        const Gemm8Maps& m = !kInt8 && job ? maps1 : maps0;
        int tm, tn, k0, k1;
        place(a, item, tm, tn, k0, k1);
        const bool narrow = gemm8_narrow(a, tn);
        const int a_row = tm * Cfg::TILE + static_cast<int>(rank) * 128, b_row = tn * Cfg::TILE + static_cast<int>(rank) * (narrow ? 64 : 128);
        // bytes of both CTAs; B across k comes in boxes of 64 columns, of which a narrow tile needs one
        const uint32_t bytes = !kInt8 && narrow ? 2 * Cfg::STAGE_BYTES - Cfg::HALF_BYTES : 2 * Cfg::STAGE_BYTES;
        for (int kb = k0; kb < k1; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag)) { fail(ERR_WAIT_EMPTY); ok = false; break; }
          uint8_t* sa = smem + stage * Cfg::STAGE_BYTES;
          uint8_t* sb = sa + Cfg::HALF_BYTES;
          if (leader) mbar_expect_tx(&full_bar[stage], bytes);   // both CTAs' bytes land on this barrier
          const uint32_t bar = map_to_cta(&full_bar[stage], 0);
          if (!kInt8 && a.a_across) {
            tma_load_2d_pair(sa, &m.a, bar, a_row, kb * BK);
            tma_load_2d_pair(sa + Cfg::HALF_BYTES / 2, &m.a, bar, a_row + 64, kb * BK);
          } else {
            tma_load_2d_pair(sa, &m.a, bar, kb * BK, a_row);
          }
          if constexpr (kInt8) {
            tma_load_2d_pair(sb, &m.b, bar, kb * BK, b_row);
          } else {
            tma_load_2d_pair(sb, &m.b, bar, b_row, kb * BK);
            if (!narrow) tma_load_2d_pair(sb + Cfg::HALF_BYTES / 2, &m.b, bar, b_row + 64, kb * BK);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    if (leader && lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      bool ok = true;
      const uint32_t base = smem_u32(smem);
      const uint64_t along_a = make_smem_desc_sw128(base, 16, 1024), along_b = make_smem_desc_sw128(base + Cfg::HALF_BYTES, 16, 1024);
      const uint64_t across_a = make_smem_desc_mn<true>(base, Cfg::HALF_BYTES / 2), across_b = make_smem_desc_mn<true>(base + Cfg::HALF_BYTES, Cfg::HALF_BYTES / 2);
      const uint32_t peer_empty0 = map_to_cta(&empty_bar[0], 1), own_empty0 = map_to_cta(&empty_bar[0], 0);
      const uint32_t peer_tfull0 = map_to_cta(&tmem_full[0], 1), own_tfull0 = map_to_cta(&tmem_full[0], 0);
      for (; ok && walk.next(jobs, job, item); ++it) {
        const Gemm8Args& a = jobs.job[kInt8 ? 0 : job];
        int tm, tn, k0, k1;
        place(a, item, tm, tn, k0, k1);
        const int width = gemm8_narrow(a, tn) ? 128 : 256;
        const bool a_across = !kInt8 && a.a_across;
        const uint64_t a0 = a_across ? across_a : along_a, b0 = kInt8 ? along_b : across_b;
        const uint32_t a_step = (a_across ? ACROSS_STEP : 32) >> 4;
        constexpr uint32_t B_STEP = (kInt8 ? 32 : ACROSS_STEP) >> 4;
        const uint32_t a_lo0 = static_cast<uint32_t>(a0), b_lo0 = static_cast<uint32_t>(b0);
        const uint64_t a_hi = a0 & 0xffffffff00000000ull, b_hi = b0 & 0xffffffff00000000ull;
        const uint32_t idesc = kInt8 ? make_idesc_i8(256, width) : make_idesc(true, 256, width, a_across, true);
        const int acc = it & 1;
        if (!mbar_wait_cluster(&tmem_empty[acc], ((it >> 1) & 1u) ^ 1u, abort_flag)) { fail(ERR_WAIT_TMEM_EMPTY); break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * Cfg::TILE;
        for (int kb = k0; kb < k1; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, abort_flag)) { fail(ERR_WAIT_FULL); ok = false; break; }
          tc_fence_after();
          const uint32_t a_lo = a_lo0 + stage * (Cfg::STAGE_BYTES >> 4), b_lo = b_lo0 + stage * (Cfg::STAGE_BYTES >> 4);
#pragma unroll
          for (int ks = 0; ks < KSTEPS; ++ks) {
            const uint64_t ad = a_hi | (a_lo + ks * a_step), bd = b_hi | (b_lo + ks * B_STEP);
            const uint32_t more = (kb > k0 || ks > 0) ? 1u : 0u;
            if constexpr (kInt8) umma_i8_pair(d_tmem, ad, bd, idesc, more);
            else umma_ss_pair<true>(d_tmem, ad, bd, idesc, more);
          }
          umma_commit_pair(own_empty0 + stage * 8);            // the stage is free in both CTAs once these have read it
          umma_commit_pair(peer_empty0 + stage * 8);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
        if (ok) {
          umma_commit_pair(own_tfull0 + acc * 8);
          umma_commit_pair(peer_tfull0 + acc * 8);
        }
      }
    }
  } else if (warp == GEMM8_PARAM_WARP) {
    // ------------------------------------------------------------ the tiles' places, scales and bias, up to two tiles ahead
    constexpr int PER_LANE = Cfg::TILE / 32;
    for (int it = 0; walk.next(jobs, job, item); ++it) {
      const Gemm8Args& a = jobs.job[kInt8 ? 0 : job];
      const int buf = it & 1;
      int tm, tn, k0, k1;
      const int part = place(a, item, tm, tn, k0, k1);
      Gemm8Place at;
      at.row0 = static_cast<long long>(tm) * Cfg::TILE + static_cast<int>(rank) * 128;
      at.out_row = static_cast<int>(at.row0) + (a.raw ? part * a.tiles_m * Cfg::TILE : 0);
      at.col0 = tn * Cfg::TILE;
      at.chunks = min(Cfg::TILE / 32, (a.N - at.col0 + 31) / 32);
      at.job = job;
      float c[PER_LANE], d[PER_LANE], r[4];
      const bool scaled = kInt8 && !a.raw;
      if (scaled) {
#pragma unroll
        for (int j = 0; j < PER_LANE; ++j) {
          const int col = at.col0 + j * 32 + lane;
          c[j] = col < a.N ? __ldg(a.col_scale + col) : 0.f;
          d[j] = (col < a.N && a.bias) ? __ldg(a.bias + col) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const long long row = at.row0 + j * 32 + lane;
          r[j] = row < a.M ? __ldg(a.row_scale + row) : 0.f;
        }
      }
      if (!mbar_wait(&param_empty[buf], ((it >> 1) & 1u) ^ 1u, abort_flag)) { fail(ERR_WAIT_EMPTY); break; }
      uint8_t* p = params + buf * Cfg::PARAM_BYTES;
      if (lane == 0) *reinterpret_cast<Gemm8Place*>(p) = at;
      if (scaled) {
        float* f = reinterpret_cast<float*>(p + 32);
#pragma unroll
        for (int j = 0; j < PER_LANE; ++j) {
          f[j * 32 + lane] = c[j];
          f[Cfg::TILE + j * 32 + lane] = d[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) f[2 * Cfg::TILE + j * 32 + lane] = r[j];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&param_full[buf]);
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs, own 128 rows of the tile)
    constexpr int G = GEMM8_EPI_WARPS / 4;
    const int quad = warp & 3, group = (warp - 2) >> 2;
    uint8_t* stage = epi + (warp - 2) * Cfg::EPI_BYTES;
    const uint32_t leader_tempty0 = map_to_cta(&tmem_empty[0], 0);
    const bool scaled = kInt8 && !jobs.job[0].raw;
    int items = 0;                                             // of this pair: the same walk, counted
    while (walk.next(jobs, job, item)) ++items;
    for (int it = 0; it < items; ++it) {
      const int acc = it & 1;
      const uint32_t parity = (it >> 1) & 1u;
      const uint8_t* p = params + acc * Cfg::PARAM_BYTES;
      if (!mbar_wait(&param_full[acc], parity, abort_flag)) { fail(ERR_WAIT_FULL); break; }
      const Gemm8Place at = *reinterpret_cast<const Gemm8Place*>(p);
      const Gemm8Args& args = jobs.job[kInt8 ? 0 : at.job];
      const CUtensorMap* tmap_out = !kInt8 && at.job ? &maps1.out : &maps0.out;
      const float* f = reinterpret_cast<const float*>(p + 32);
      const float rs = scaled ? f[2 * Cfg::TILE + quad * 32 + lane] : 0.f;
      const long long row0 = at.row0 + quad * 32;
      const int chunks = row0 < args.M ? at.chunks : 0;        // warp-uniform
      if (!mbar_wait(&tmem_full[acc], parity, abort_flag)) { fail(ERR_WAIT_TMEM_FULL); break; }
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * Cfg::TILE;
      // 16 columns at a time, the next 16 on their way from tensor memory meanwhile
      uint32_t r0[16], r1[16];
      __syncwarp();
      if (group < chunks) tmem_ld_32x16(taddr + group * 32, r0);
#pragma unroll 1   // one copy of the code: it has to stay in the instruction cache
      for (int c = group; c < chunks; c += G) {
        const float* cs = f + c * 32;
        const int col0 = at.col0 + c * 32;
        tmem_ld_wait();
        tmem_ld_32x16(taddr + c * 32 + 16, r1);
        if (scaled) gemm8_finish(r0, rs, cs, cs + Cfg::TILE, args.act);
        gemm8_write(args, tmap_out, r0, stage, row0, at.out_row + quad * 32, col0, 0, lane);
        __syncwarp();
        tmem_ld_wait();
        if (c + G < chunks) tmem_ld_32x16(taddr + (c + G) * 32, r0);
        if (scaled) gemm8_finish(r1, rs, cs + 16, cs + Cfg::TILE + 16, args.act);
        gemm8_write(args, tmap_out, r1, stage, row0, at.out_row + quad * 32, col0 + 16, 1, lane);
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(leader_tempty0 + acc * 8);
      __syncwarp();
      if (lane == 0) mbar_arrive(&param_empty[acc]);
    }
    if (lane == 0) tma_store_wait_all<0>();
  }

  // ---------------------------------------------------------------- teardown
  if (*abort_flag) {
    for (int i = 0; i < 100; ++i) __nanosleep(10000);          // let copies and MMAs in flight land (about 1 ms)
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();                                              // neither CTA frees TMEM or exits while the other still uses it
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
}

// Adds the parts of a product split along k, in order, and applies the epilogue to 4 columns.
template <bool kInt8>
__device__ __forceinline__ void gemm8_join(const Gemm8Args& a, const uint32_t* ws, long long ld_ws, long long plane, long long row, int col) {
  const uint4* src = reinterpret_cast<const uint4*>(ws + row * ld_ws + col);
  float v[4];
  if constexpr (kInt8) {
    int s[4] = {0, 0, 0, 0};
#pragma unroll 4
    for (int p = 0; p < a.splits; ++p) {
      const uint4 t = src[p * (plane / 4)];
      s[0] += static_cast<int>(t.x); s[1] += static_cast<int>(t.y); s[2] += static_cast<int>(t.z); s[3] += static_cast<int>(t.w);
    }
    const float rs = __ldg(a.row_scale + row);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = col + j < a.N;
      v[j] = gemm8_act(fmaf(static_cast<float>(s[j]) * rs, in ? __ldg(a.col_scale + col + j) : 0.f, (in && a.bias) ? __ldg(a.bias + col + j) : 0.f), a.act);
    }
  } else {
    v[0] = v[1] = v[2] = v[3] = 0.f;
#pragma unroll 4
    for (int p = 0; p < a.splits; ++p) {
      const uint4 t = src[p * (plane / 4)];
      v[0] += __uint_as_float(t.x); v[1] += __uint_as_float(t.y); v[2] += __uint_as_float(t.z); v[3] += __uint_as_float(t.w);
    }
  }
  const long long at = row * a.ld_out + col;
  if (a.wide_store && col + 4 <= a.N) {
    if (a.out_bf16) *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) = make_uint2(F2(v[0], v[1]).bf16(), F2(v[2], v[3]).bf16());
    else *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (col + j < a.N) {
      if (a.out_bf16) static_cast<__nv_bfloat16*>(a.out)[at + j] = __float2bfloat16(v[j]);
      else static_cast<float*>(a.out)[at + j] = v[j];
    }
  }
}
// What the tensor-core launch left to be added up: the parts of its products (those with splits > 1), and in the blocks from
// sum_at on the column sums, 32 columns per block of 512 threads.
struct Gemm8Finish {
  Gemm8Args job[2];
  const uint32_t* ws[2];
  long long ld_ws[2], plane[2], pieces[2];   // pieces of 4 columns; 0: nothing to join
  Divisor per_row[2];
  unsigned sum_at;
  const float* partial;
  float* sums;
  int blocks, F;
};
template <bool kInt8>
__global__ void __launch_bounds__(512) gemm8_finish_kernel(const __grid_constant__ Gemm8Finish f) {
  __shared__ float part[16][33];
  wait_for_previous_kernel();
  if (blockIdx.x >= f.sum_at) {
    column_total(f.partial, f.sums, f.blocks, f.F, static_cast<int>(blockIdx.x - f.sum_at), part);
    return;
  }
#pragma unroll
  for (int j = 0; j < (kInt8 ? 1 : 2); ++j) {
    for (long long i = blockIdx.x * 512ll + threadIdx.x; i < f.pieces[j]; i += f.sum_at * 512ll) {
      long long row;
      if (f.pieces[j] < (1ll << 31)) row = f.per_row[j].quotient(static_cast<int>(i));
      else row = i / f.per_row[j].d;
      gemm8_join<kInt8>(f.job[j], f.ws[j], f.ld_ws[j], f.plane[j], row, static_cast<int>(i - row * f.per_row[j].d) * 4);
    }
  }
}

}  // namespace gb
