// Matrix products of the 8-bit row operators on the tensor cores: C[M][N] = epilogue(sum over k of A(m, k) B(n, k)).
//
//   Gemm8Kind::Q8      A = x_q [M][K], B = W_q [N][K], int8 along k (kind::i8, exact int32 sums): linear_q8
//   Gemm8Kind::DGRAD   A = grad_out [M][k] along k, B = W [k][N] across k (bf16, fp32 sums): grad_x = grad_out W
//   Gemm8Kind::WGRAD   A = grad_out [k][M], B = x [k][N], both across k (bf16): grad_W = grad_out^T x
//
// A pair of CTAs shares one tcgen05.mma (cta_group::2): a 256 x 256 tile of C, of which each CTA loads 128 rows of A and
// 128 of B per k-block of 128 bytes and keeps 128 rows of the accumulator in its own tensor memory, twice, so that one
// tile is written while the next is computed. Roles per CTA: warp 0 TMA producer (own halves, bytes counted on the
// leader's barrier), warp 1 MMA issuer (leader) and TMEM allocation, the rest epilogue. Every wait is bounded and reports
// through the device status word. Nothing is broadcast by TMA.
//
// Few tiles of a long product are split along k: every part stores its raw 32-bit sums to its own plane of a workspace and
// a second kernel adds the planes in order (no atomics: results repeat bit for bit).
#pragma once
#include "ptx.cuh"
#include <cuda_bf16.h>

namespace gb {

enum class Gemm8Kind { Q8, DGRAD, WGRAD };

struct Gemm8Args {
  long long M;
  int N;
  int tiles_m, tiles_n, tile_group, k_blocks;
  int splits, k_per_split;    // k-blocks per part
  // epilogue
  void* out;                  // C [M][N] fp32 or bf16, or the workspace [splits][M][ld_out] of raw sums
  long long ld_out;
  int out_bf16, raw;
  int wide_store;             // rows of C start on 4-element boundaries
  const float* row_scale;     // Q8: per row and per column, and the bias
  const float* col_scale;
  const float* bias;
  int act;
  int* err;
};

constexpr int GEMM8_EPI_WARPS = 8;
constexpr int GEMM8_THREADS = 64 + 32 * GEMM8_EPI_WARPS;

struct Gemm8Cfg {
  static constexpr int TILE = 256;
  static constexpr int HALF_BYTES = 128 * 128;               // 128 rows (or columns) x 128 bytes
  static constexpr int STAGE_BYTES = 2 * HALF_BYTES;
  static constexpr int STAGES = 6;
  static constexpr int EPI_BYTES = 32 * 128;                 // per epilogue warp: 32 rows x 32 columns of 32 bits
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + GEMM8_EPI_WARPS * EPI_BYTES + 1024 /*align slack*/ + 256 /*barriers*/;
  static constexpr int TMEM_COLS = 512;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory of one CTA");
};

// ---- epilogue arithmetic
__device__ __forceinline__ float gemm8_act(float v, int act) {
  // GELU (tanh form) as v * sigmoid(2 u): one exponential and one division, accurate for v far below zero too
  switch (act) {
    case 1: return __fdividef(v, 1.f + __expf(-2.f * 0.7978845608028654f * v * fmaf(0.044715f, v * v, 1.f)));
    case 2: return __fdividef(v, 1.f + __expf(-v));
    case 3: return v < 0.f ? 0.f : v;
    default: return v;
  }
}

// Tile of the persistent loop: `fast` blocks are walked in groups so that the tiles of one moment share rows of A and B.
static __device__ __noinline__ uint64_t gemm8_tile(int tile, int num_fast, int num_slow, int group) {
  const int per_group = group * num_slow;
  const int g = tile / per_group, first = g * group;
  const int size = min(num_fast - first, group), r = tile - g * per_group, slow = r / size;
  return static_cast<uint64_t>(static_cast<uint32_t>(first + r - slow * size)) | (static_cast<uint64_t>(static_cast<uint32_t>(slow)) << 32);
}

// Writes 32 rows x 32 columns. They lie in shared memory as raw 32-bit sums, row r at 128 r with its 16-byte pieces
// exchanged by r % 8 (no bank conflicts on either side). W columns per lane: 4 where rows of C are aligned for it, else 1;
// either way the lanes of one store cover whole pieces of rows.
template <Gemm8Kind KIND, int W>
__device__ __forceinline__ void gemm8_store_block(const Gemm8Args& a, const uint8_t* stage, long long row0, int col0, int lane, uint8_t* out_base) {
  constexpr int PER_ROW = 32 / W;            // lanes per row
  constexpr int ROWS = 32 / PER_ROW;         // rows per store
  const int piece = (lane % PER_ROW) * W;    // first column of the lane
  const int col = col0 + piece;
  if (col >= a.N) return;
  float cs[W], bias[W];
  if constexpr (KIND == Gemm8Kind::Q8) {
    if (!a.raw) {
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const bool in = col + j < a.N;
        cs[j] = in ? __ldg(a.col_scale + col + j) : 0.f;
        bias[j] = (in && a.bias) ? __ldg(a.bias + col + j) : 0.f;
      }
    }
  }
#pragma unroll 8
  for (int i = 0; i < 32 / ROWS; ++i) {
    const int r = i * ROWS + lane / PER_ROW;
    const long long row = row0 + r;
    if (row >= a.M) break;
    uint32_t w[W];
    const uint8_t* src = stage + r * 128 + (((piece >> 2) ^ (r & 7)) << 4) + (piece & 3) * 4;
    if constexpr (W == 4) {
      const uint4 t = *reinterpret_cast<const uint4*>(src);
      w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(src);
    }
    const long long at = row * a.ld_out + col;
    if (a.raw) {                             // the workspace's rows are multiples of 4 long
      if constexpr (W == 4) *reinterpret_cast<uint4*>(out_base + at * 4) = make_uint4(w[0], w[1], w[2], w[3]);
      else *reinterpret_cast<uint32_t*>(out_base + at * 4) = w[0];
      continue;
    }
    float v[W];
    if constexpr (KIND == Gemm8Kind::Q8) {
      const float rs = __ldg(a.row_scale + row);
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = gemm8_act(fmaf(static_cast<float>(static_cast<int>(w[j])) * rs, cs[j], bias[j]), a.act);
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = __uint_as_float(w[j]);
    }
    if (a.out_bf16) {
      __nv_bfloat16* p = reinterpret_cast<__nv_bfloat16*>(out_base) + at;
      if constexpr (W == 4) {
        if (col + 4 <= a.N) {
          const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
          *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
          continue;
        }
      }
#pragma unroll
      for (int j = 0; j < W; ++j)
        if (col + j < a.N) p[j] = __float2bfloat16(v[j]);
    } else {
      float* p = reinterpret_cast<float*>(out_base) + at;
      if constexpr (W == 4) {
        if (col + 4 <= a.N) {
          *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
          continue;
        }
      }
#pragma unroll
      for (int j = 0; j < W; ++j)
        if (col + j < a.N) p[j] = v[j];
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

template <Gemm8Kind KIND>
__global__ void __launch_bounds__(GEMM8_THREADS, 1)
gemm8_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const Gemm8Args args) {
  using Cfg = Gemm8Cfg;
  constexpr int STAGES = Cfg::STAGES;
  constexpr bool kInt8 = KIND == Gemm8Kind::Q8, kAMn = KIND == Gemm8Kind::WGRAD, kBMn = KIND != Gemm8Kind::Q8;
  constexpr int BK = kInt8 ? 128 : 64;                         // k per stage
  constexpr int KSTEPS = 4;                                    // instructions per stage, 32 bytes of k each
  constexpr uint32_t MN_STEP = 16 * 128;                       // bytes of an operand across k per instruction
  constexpr uint32_t IDESC = kInt8 ? make_idesc_i8(256, 256) : make_idesc(true, 256, 256, kAMn, kBMn);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + STAGES * Cfg::STAGE_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(epi + GEMM8_EPI_WARPS * Cfg::EPI_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tmem_full = empty_bar + STAGES;
  uint64_t* tmem_empty = tmem_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();                     // 0 = leader
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int tiles = args.tiles_m * args.tiles_n, items = tiles * args.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);                              // used in the leader only
      mbar_init(&empty_bar[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tmem_full[i], 1);
      mbar_init(&tmem_empty[i], 2 * GEMM8_EPI_WARPS);          // used in the leader only
    }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_b);
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

  // a failed wait stops both CTAs: the peer's waits poll its own flag
  auto fail = [&](int code) {
    if (!*abort_flag) atomicCAS(args.err, 0, code);
    *abort_flag = 1;
    st_cluster_u32(map_to_cta(const_cast<int*>(abort_flag), rank ^ 1u), 1u);
  };
  auto k_range = [&](int item, int& k0, int& k1) {
    const int part = item / tiles;
    k0 = part * args.k_per_split;
    k1 = min(args.k_blocks, k0 + args.k_per_split);
    return item - part * tiles;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs, own halves)
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int item = pair; item < items && ok; item += num_pairs) {
        int k0, k1;
        const uint64_t t = gemm8_tile(k_range(item, k0, k1), args.tiles_m, args.tiles_n, args.tile_group);
        const int a_row = static_cast<int>(static_cast<uint32_t>(t)) * Cfg::TILE + static_cast<int>(rank) * 128;
        const int b_row = static_cast<int>(t >> 32) * Cfg::TILE + static_cast<int>(rank) * 128;
        for (int kb = k0; kb < k1; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag)) { fail(ERR_WAIT_EMPTY); ok = false; break; }
          uint8_t* sa = smem + stage * Cfg::STAGE_BYTES;
          uint8_t* sb = sa + Cfg::HALF_BYTES;
          if (leader) mbar_expect_tx(&full_bar[stage], 2 * Cfg::STAGE_BYTES);   // both CTAs' bytes land on this barrier
          const uint32_t bar = map_to_cta(&full_bar[stage], 0);
          if constexpr (kAMn) {
            tma_load_2d_pair(sa, &tmap_a, bar, a_row, kb * BK);
            tma_load_2d_pair(sa + Cfg::HALF_BYTES / 2, &tmap_a, bar, a_row + 64, kb * BK);
          } else {
            tma_load_2d_pair(sa, &tmap_a, bar, kb * BK, a_row);
          }
          if constexpr (kBMn) {
            tma_load_2d_pair(sb, &tmap_b, bar, b_row, kb * BK);
            tma_load_2d_pair(sb + Cfg::HALF_BYTES / 2, &tmap_b, bar, b_row + 64, kb * BK);
          } else {
            tma_load_2d_pair(sb, &tmap_b, bar, kb * BK, b_row);
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
      const uint64_t a0 = kAMn ? make_smem_desc_mn<true>(base, Cfg::HALF_BYTES / 2) : make_smem_desc_sw128(base, 16, 1024);
      const uint64_t b0 = kBMn ? make_smem_desc_mn<true>(base + Cfg::HALF_BYTES, Cfg::HALF_BYTES / 2) : make_smem_desc_sw128(base + Cfg::HALF_BYTES, 16, 1024);
      const uint32_t a_lo0 = static_cast<uint32_t>(a0), b_lo0 = static_cast<uint32_t>(b0);
      const uint64_t a_hi = a0 & 0xffffffff00000000ull, b_hi = b0 & 0xffffffff00000000ull;
      constexpr uint32_t A_STEP = (kAMn ? MN_STEP : 32) >> 4, B_STEP = (kBMn ? MN_STEP : 32) >> 4;
      const uint32_t peer_empty0 = map_to_cta(&empty_bar[0], 1), own_empty0 = map_to_cta(&empty_bar[0], 0);
      const uint32_t peer_tfull0 = map_to_cta(&tmem_full[0], 1), own_tfull0 = map_to_cta(&tmem_full[0], 0);
      for (int item = pair; item < items && ok; item += num_pairs, ++it) {
        int k0, k1;
        k_range(item, k0, k1);
        const int acc = it & 1;
        if (!mbar_wait(&tmem_empty[acc], ((it >> 1) & 1u) ^ 1u, abort_flag)) { fail(ERR_WAIT_TMEM_EMPTY); break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * Cfg::TILE;
        for (int kb = k0; kb < k1; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, abort_flag)) { fail(ERR_WAIT_FULL); ok = false; break; }
          tc_fence_after();
          const uint32_t a_lo = a_lo0 + stage * (Cfg::STAGE_BYTES >> 4), b_lo = b_lo0 + stage * (Cfg::STAGE_BYTES >> 4);
#pragma unroll
          for (int ks = 0; ks < KSTEPS; ++ks) {
            const uint64_t ad = a_hi | (a_lo + ks * A_STEP), bd = b_hi | (b_lo + ks * B_STEP);
            const uint32_t more = (kb > k0 || ks > 0) ? 1u : 0u;
            if constexpr (kInt8) umma_i8_pair(d_tmem, ad, bd, IDESC, more);
            else umma_ss_pair<true>(d_tmem, ad, bd, IDESC, more);
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
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs, own 128 rows of the tile)
    constexpr int NCHUNK = Cfg::TILE / 32, G = GEMM8_EPI_WARPS / 4;
    const int quad = warp & 3, group = (warp - 2) >> 2;
    uint8_t* stage = epi + (warp - 2) * Cfg::EPI_BYTES;
    const uint32_t leader_tempty0 = map_to_cta(&tmem_empty[0], 0);
    int it = 0;
    for (int item = pair; item < items; item += num_pairs, ++it) {
      int k0, k1;
      const int tile = k_range(item, k0, k1);
      const uint64_t t = gemm8_tile(tile, args.tiles_m, args.tiles_n, args.tile_group);
      const long long row0 = static_cast<long long>(static_cast<uint32_t>(t)) * Cfg::TILE + static_cast<int>(rank) * 128 + quad * 32;
      const int first_col = static_cast<int>(t >> 32) * Cfg::TILE;
      uint8_t* out = static_cast<uint8_t*>(args.out);
      if (args.raw) out += static_cast<long long>(item / tiles) * args.M * args.ld_out * 4;
      const int acc = it & 1;
      if (!mbar_wait(&tmem_full[acc], (it >> 1) & 1u, abort_flag)) { fail(ERR_WAIT_TMEM_FULL); break; }
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * Cfg::TILE;
      for (int c = group; c < NCHUNK; c += G) {
        const int col0 = first_col + c * 32;
        if (col0 >= args.N || row0 >= args.M) break;           // warp-uniform
        uint32_t r[32];
        __syncwarp();
        tmem_ld_32x32(taddr + c * 32, r);
        tmem_ld_wait();
#pragma unroll
        for (int p = 0; p < 8; ++p)
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((p ^ (lane & 7)) << 4)) = make_uint4(r[4 * p], r[4 * p + 1], r[4 * p + 2], r[4 * p + 3]);
        __syncwarp();
        if (args.wide_store) gemm8_store_block<KIND, 4>(args, stage, row0, col0, lane, out);
        else gemm8_store_block<KIND, 1>(args, stage, row0, col0, lane, out);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(leader_tempty0 + acc * 8);
    }
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

// Adds the parts of a product split along k, in order, and applies the epilogue. Four columns per thread.
template <Gemm8Kind KIND>
__global__ void __launch_bounds__(256) gemm8_join_kernel(const Gemm8Args a, const uint32_t* __restrict__ ws, long long ld_ws) {
  const int per_row = (a.N + 3) / 4;
  const long long total = a.M * per_row, plane = a.M * ld_ws;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long row = i / per_row;
    const int col = static_cast<int>(i - row * per_row) * 4;
    const uint4* src = reinterpret_cast<const uint4*>(ws + row * ld_ws + col);
    float v[4];
    if constexpr (KIND == Gemm8Kind::Q8) {
      int s[4] = {0, 0, 0, 0};
#pragma unroll 4
      for (int p = 0; p < a.splits; ++p) {
        const uint4 t = __ldg(src + p * (plane / 4));
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
        const uint4 t = __ldg(src + p * (plane / 4));
        v[0] += __uint_as_float(t.x); v[1] += __uint_as_float(t.y); v[2] += __uint_as_float(t.z); v[3] += __uint_as_float(t.w);
      }
    }
    const long long at = row * a.ld_out + col;
    if (a.wide_store && col + 4 <= a.N) {
      if (a.out_bf16) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      } else {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
      }
      continue;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (col + j < a.N) {
        if (a.out_bf16) static_cast<__nv_bfloat16*>(a.out)[at + j] = __float2bfloat16(v[j]);
        else static_cast<float*>(a.out)[at + j] = v[j];
      }
    }
  }
}

}  // namespace gb
