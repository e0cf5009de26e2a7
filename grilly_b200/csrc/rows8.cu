// Rows in 8 bits: quantise, read back, RMSNorm with the residual's addition into 8-bit rows, and that norm's backward
// pass from the 8-bit checkpoint of its input. The definitions stand with the entry points in include/grilly_b200.h.
//
// All of them are bound by HBM. A persistent CTA of 512 threads per SM works on several rows at a time, a team of 32 to 512
// threads on each (32 values per thread). Every team has a ring of rows in shared memory that bulk copies fill several rows
// ahead, so that memory is read all the time and not only while a block has nothing else to do (blocks that each load,
// reduce and store a row reached half the bandwidth). A row goes from there into registers, is reduced once and written once.
// Rows that start off 16-byte boundaries (odd lengths) are copied from the boundary below and read value by value.
#include "rows8.h"
#include "rows8_sum.cuh"
#include "ptx.cuh"
#include <cuda_bf16.h>
#include <algorithm>
#include <initializer_list>

namespace gb {
namespace {

constexpr int PER_THREAD = 32;         // values of a row per thread
constexpr int CTA = 512;
constexpr int MAX_TEAMS = CTA / 32;
constexpr int MAX_DEPTH = 8;           // rows in a team's ring
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
    g[0] = gamma[col];
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 4) {
      const float4 t = *reinterpret_cast<const float4*>(gamma + col + j);
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

// ---- the ring
// Up to three row tensors (all 16-byte aligned) and the geometry that the host chose.
struct Ring {
  const void* src[3];
  long long pitch[3];        // bytes from row to row in memory
  long long total[3];        // bytes of the tensor
  int bytes[3];              // bytes of one row
  int at[3];                 // where a tensor's row lies in a slot
  int tensors, slot;         // slot: bytes, a multiple of 16
  int team, teams, depth;    // threads per team, teams per CTA, slots per team
  int gamma_at, slots_at;    // offsets in shared memory: barriers first, then reductions, gamma, slots
  long long rows;
  long long first_tail;      // from this row on, bytes past the tensors' last 16-byte boundary are needed
  int F;
  int* err;
};
struct RowStats {
  float sq;
  uint32_t my, mh;
};
constexpr int RED_AT = MAX_TEAMS * MAX_DEPTH * 8;              // RowStats [2][CTA / 32]
constexpr int ABORT_AT = RED_AT + 2 * (CTA / 32) * 12;
constexpr int GAMMA_AT = (ABORT_AT + 4 + 15) / 16 * 16;

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// A team's view of the ring. All of a team's threads call next() and done() together.
struct Team {
  const Ring& g;
  uint8_t* smem;
  uint64_t* bars;
  volatile int* abort_flag;
  int team, tid, slot, parity;   // parity: of the slot's barrier
  uint32_t flip;                 // which half of the reduction scratch
  long long row, step;

  __device__ Team(const Ring& ring, uint8_t* shared) : g(ring), smem(shared), flip(0) {
    team = threadIdx.x / g.team;
    tid = threadIdx.x - team * g.team;
    bars = reinterpret_cast<uint64_t*>(smem) + team * g.depth;
    abort_flag = reinterpret_cast<volatile int*>(smem + ABORT_AT);
    row = team < g.teams ? static_cast<long long>(team) * gridDim.x + blockIdx.x : g.rows;   // long rows leave threads idle
    step = static_cast<long long>(g.teams) * gridDim.x;
    slot = 0;
    parity = 0;
  }
  // whole CTA: barriers, gamma, the first rows on their way
  __device__ void start(const float* gamma) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < g.teams * g.depth; ++i) mbar_init(reinterpret_cast<uint64_t*>(smem) + i, 1);
      *abort_flag = 0;
      fence_mbar_init();
    }
    __syncthreads();
    if (tid == 0) {
      for (int d = 0; d < g.depth; ++d) fetch(row + d * step, d);
    }
    float* gm = reinterpret_cast<float*>(smem + g.gamma_at);
    if (gamma)
      for (int c = threadIdx.x; c < g.F; c += CTA) gm[c] = __ldg(gamma + c);
    __syncthreads();
  }
  // the aligned bytes [from, to) of row r of tensor i that a copy brings, relative to the tensor
  __device__ void span(int i, long long r, long long& from, long long& to) const {
    from = r * g.pitch[i] & ~15ll;
    to = min((r * g.pitch[i] + g.bytes[i] + 15) & ~15ll, g.total[i] & ~15ll);
    if (to < from) to = from;
  }
  __device__ uint8_t* slot_of(int d) const { return smem + g.slots_at + (team * g.depth + d) * g.slot; }
  __device__ void fetch(long long r, int d) const {
    if (r >= g.rows) return;
    uint32_t sum = 0;
    long long from[3], to[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (i < g.tensors) {
        span(i, r, from[i], to[i]);
        sum += static_cast<uint32_t>(to[i] - from[i]);
      }
    }
    mbar_expect_tx(&bars[d], sum);
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < g.tensors && to[i] > from[i])
        bulk_load(slot_of(d) + g.at[i], static_cast<const uint8_t*>(g.src[i]) + from[i], static_cast<uint32_t>(to[i] - from[i]), &bars[d]);
  }
  __device__ void sync() const {
    if (g.team == 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(g.team) : "memory");
  }
  // waits for the current row; false: the wait ran out (reported) and the team stops
  __device__ bool next() {
    int ok = mbar_wait(&bars[slot], static_cast<uint32_t>(parity), abort_flag) ? 1 : 0;
    if (!ok) {
      if (!*abort_flag) atomicCAS(g.err, 0, ERR_WAIT_FULL);
      *abort_flag = 1;
    }
    if (row >= g.first_tail) {
      // the last bytes of a tensor that ends off a 16-byte boundary are not copied in bulk
      for (int i = 0; i < g.tensors; ++i) {
        long long from, to;
        span(i, row, from, to);
        const long long end = row * g.pitch[i] + g.bytes[i], first = max(to, row * g.pitch[i]);
        if (tid < end - first) {
          const long long at = first + tid;
          slot_of(slot)[g.at[i] + (at - from)] = static_cast<const uint8_t*>(g.src[i])[at];
        }
      }
    }
    if (g.team == 32) {
      ok = __all_sync(FULL, ok);
    } else {
      asm volatile(
          "{\n\t"
          ".reg .pred p, q;\n\t"
          "setp.ne.s32 p, %1, 0;\n\t"
          "bar.red.and.pred q, %2, %3, p;\n\t"
          "selp.s32 %0, 1, 0, q;\n\t"
          "}\n"
          : "=r"(ok) : "r"(ok), "r"(team + 1), "r"(g.team) : "memory");
    }
    return ok != 0;
  }
  // the current row of tensor i: its first value
  template <class T>
  __device__ const T* values(int i) const {
    return reinterpret_cast<const T*>(slot_of(slot) + g.at[i] + static_cast<int>(row * g.pitch[i] & 15));
  }
  // everything of the row has been read
  __device__ void done() {
    sync();
    if (tid == 0) fetch(row + g.depth * step, slot);
    row += step;
    if (++slot == g.depth) {
      slot = 0;
      parity ^= 1;
    }
  }
  // whole CTA, after the last row: copies that a failed wait left in flight get time to land (about 1 ms)
  __device__ void end() const {
    __syncthreads();
    if (*abort_flag)
      for (int i = 0; i < 100; ++i) __nanosleep(10000);
  }
  // over the team, in an order that its size alone decides
  template <bool kSum, bool kMax, bool kTwo>
  __device__ RowStats reduce(RowStats s) {
    if constexpr (kSum) s.sq = warp_sum(s.sq);
    if constexpr (kMax) s.mh = warp_max(s.mh);
    if constexpr (kTwo) s.my = warp_max(s.my);
    if (g.team > 32) {
      const int lane = threadIdx.x & 31, warps = g.team >> 5;
      RowStats* red = reinterpret_cast<RowStats*>(smem + RED_AT) + flip * (CTA / 32);
      flip ^= 1;             // the other half is free again once every thread has passed this row's barriers
      if (lane == 0) red[threadIdx.x >> 5] = s;
      sync();
      s = lane < warps ? red[team * warps + lane] : RowStats{0.f, 0u, 0u};
      if constexpr (kSum) s.sq = warp_sum(s.sq);
      if constexpr (kMax) s.mh = warp_max(s.mh);
      if constexpr (kTwo) s.my = warp_max(s.my);
    }
    return s;
  }
};
#define FOR_PIECES(i, c) _Pragma("unroll") for (int i = 0, c = t.tid * VEC; i < NV; ++i, c += t.g.team * VEC) if (c < F)

// ---- a row per block of 1024 threads, for what the ring does not take
__device__ __forceinline__ RowStats block_reduce(RowStats s, RowStats* red) {
  const int lane = threadIdx.x & 31;
  s.sq = warp_sum(s.sq);
  s.mh = warp_max(s.mh);
  s.my = warp_max(s.my);
  if (lane == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = red[lane];
  s.sq = warp_sum(s.sq);
  s.mh = warp_max(s.mh);
  s.my = warp_max(s.my);
  return s;
}

// ---------------------------------------------------------------- quantise
template <class T, int VEC>
__global__ void __launch_bounds__(CTA, 1) quantize_rows_kernel(const __grid_constant__ Ring ring, int8_t* q, float* scale, long long ld) {
  constexpr int NV = PER_THREAD / VEC;
  extern __shared__ __align__(16) uint8_t smem[];
  Team t(ring, smem);
  t.start(nullptr);
  const int F = ring.F;
  for (; t.row < ring.rows; t.done()) {
    if (!t.next()) break;
    const T* xp = t.values<T>(0);
    float v[NV][VEC];
    RowStats s{0.f, 0u, 0u};
    FOR_PIECES(i, c) {
      load_vec(xp + c, v[i]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) s.mh = max(s.mh, abs_bits(v[i][j]));
    }
    s = t.reduce<false, true, false>(s);
    const float sc = row_scale(s.mh), inv = row_inverse(sc);
    const uint32_t keep = s.mh >= INF_BITS ? 0u : FULL;
    int8_t* qp = q + t.row * ld;
    FOR_PIECES(i, c) store_q(qp + c, v[i], inv, keep);
    for (long long c = F + t.tid; c < ld; c += ring.team) qp[c] = 0;
    if (t.tid == 0) scale[t.row] = sc;
  }
  t.end();
}
// Rows too long for the ring, or off 16-byte boundaries from the first: a block per row, read twice.
template <class T>
__global__ void __launch_bounds__(1024) quantize_long_rows_kernel(const T* x, int8_t* q, float* scale, long long rows, int F, long long ld) {
  __shared__ RowStats red[32];
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xp = x + row * F;
    RowStats s{0.f, 0u, 0u};
    float v[1];
    for (int c = threadIdx.x; c < F; c += blockDim.x) {
      load_vec(xp + c, v);
      s.mh = max(s.mh, abs_bits(v[0]));
    }
    s = block_reduce(s, red);
    const float sc = row_scale(s.mh), inv = row_inverse(sc);
    const uint32_t keep = s.mh >= INF_BITS ? 0u : FULL;
    for (long long c = threadIdx.x; c < ld; c += blockDim.x) {
      v[0] = 0.f;
      if (c < F) load_vec(xp + c, v);
      store_q(q + row * ld + c, v, inv, keep);
    }
    if (threadIdx.x == 0) scale[row] = sc;
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
  const int lane = threadIdx.x & 31;
  for (long long row = blockIdx.x * 8ll + (threadIdx.x >> 5); row < rows; row += gridDim.x * 8ll) {
    const float s = __ldg(scale + row);
#pragma unroll 8
    for (int c = lane; c < F; c += 32) {
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
// max |h| are taken together and nothing waits for rstd. A row has been read whole before h is written (in place).
template <class T, int VEC>
__global__ void __launch_bounds__(CTA, 1) rmsnorm_q8_kernel(const __grid_constant__ Ring ring, const NormQ8Args a) {
  constexpr int NV = PER_THREAD / VEC;
  extern __shared__ __align__(16) uint8_t smem[];
  Team t(ring, smem);
  t.start(a.gamma);
  const float* gamma = a.gamma ? reinterpret_cast<const float*>(smem + ring.gamma_at) : nullptr;
  const int F = ring.F;
  const float inv_f = 1.f / static_cast<float>(F);
  for (; t.row < ring.rows; t.done()) {
    if (!t.next()) break;
    const T* xp = t.values<T>(0);
    const T* rp = ring.tensors > 1 ? t.values<T>(1) : nullptr;
    float h[NV][VEC], sum[4] = {0.f, 0.f, 0.f, 0.f};
    RowStats s{0.f, 0u, 0u};
    FOR_PIECES(i, c) {
      load_vec(xp + c, h[i]);
      if (rp) {
        float r[VEC];
        load_vec(rp + c, r);
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[i][j] += r[j];
      }
      float gm[VEC];
      load_gamma(gamma, c, gm);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float& acc = sum[(i * VEC + j) & 3];
        acc = fmaf(h[i][j], h[i][j], acc);
        s.my = max(s.my, abs_bits(h[i][j] * gm[j]));
        s.mh = max(s.mh, abs_bits(h[i][j]));
      }
    }
    s.sq = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    s = t.reduce<true, true, true>(s);
    const NormScales r = norm_scales(s, inv_f, a.eps);
    T* hp = a.h ? static_cast<T*>(a.h) + t.row * F : nullptr;
    int8_t* yq = a.yq + t.row * a.ld;
    int8_t* hq = a.hq ? a.hq + t.row * a.ld : nullptr;
    FOR_PIECES(i, c) {
      if (hp) store_vec(hp + c, h[i]);
      if (hq) store_q(hq + c, h[i], r.hi, r.keep);
      float gm[VEC];
      load_gamma(gamma, c, gm);
#pragma unroll
      for (int j = 0; j < VEC; ++j) gm[j] *= h[i][j] * r.rstd;
      store_q(yq + c, gm, r.yi, r.keep);
    }
    for (long long c = F + t.tid; c < a.ld; c += ring.team) {
      yq[c] = 0;
      if (hq) hq[c] = 0;
    }
    if (t.tid == 0) norm_row_done(a, r, t.row);
  }
  t.end();
}
// The same a row per block, read twice, h written as it is read again.
template <class T>
__global__ void __launch_bounds__(1024) rmsnorm_q8_long_kernel(const NormQ8Args a) {
  __shared__ RowStats red[32];
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
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
    for (int c = threadIdx.x; c < a.F; c += blockDim.x) {
      in(c);
      s.sq = fmaf(h[0], h[0], s.sq);
      s.my = max(s.my, abs_bits(h[0] * gm[0]));
      s.mh = max(s.mh, abs_bits(h[0]));
    }
    s = block_reduce(s, red);
    const NormScales n = norm_scales(s, 1.f / static_cast<float>(a.F), a.eps);
    for (long long c = threadIdx.x; c < a.ld; c += blockDim.x) {
      h[0] = gm[0] = 0.f;
      if (c < a.F) {
        in(static_cast<int>(c));
        if (a.h) store_vec(static_cast<T*>(a.h) + row * a.F + c, h);
      }
      if (a.hq) store_q(a.hq + row * a.ld + c, h, n.hi, n.keep);
      gm[0] *= h[0] * n.rstd;
      store_q(a.yq + row * a.ld + c, gm, n.yi, n.keep);
    }
    if (threadIdx.x == 0) norm_row_done(a, n, row);
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
  int F;
};

// A thread keeps the same columns of every row that its team meets, so the gradient of gamma is summed in registers and
// leaves once per CTA; the CTAs' sums are added by sum_partials_kernel in a fixed order. The row is read from the ring
// twice (before and after its one sum) instead of being held next to those sums.
template <class T, int VEC>
__global__ void __launch_bounds__(CTA, 1) rmsnorm_bwd_kernel(const __grid_constant__ Ring ring, const NormBwdQ8Args a) {
  constexpr int NV = PER_THREAD / VEC;
  extern __shared__ __align__(16) uint8_t smem[];
  Team t(ring, smem);
  t.start(a.gamma);
  const float* gamma = a.gamma ? reinterpret_cast<const float*>(smem + ring.gamma_at) : nullptr;
  const int F = ring.F;
  const float inv_f = 1.f / static_cast<float>(F);
  float acc[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[i][j] = 0.f;
  for (; t.row < ring.rows; t.done()) {
    const float rstd = __ldg(a.rstd + t.row), s = __ldg(a.hs + t.row) * rstd;
    if (!t.next()) break;
    const int8_t* qp = t.values<int8_t>(0);
    const T* gp = t.values<T>(1);
    const T* rp = ring.tensors > 2 ? t.values<T>(2) : nullptr;
    float dots[4] = {0.f, 0.f, 0.f, 0.f};
    FOR_PIECES(i, c) {
      float g[VEC], n[VEC], gm[VEC];
      load_vec(gp + c, g);
      load_q(qp + c, n);
      load_gamma(gamma, c, gm);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        n[j] *= s;
        acc[i][j] = fmaf(g[j], n[j], acc[i][j]);
        float& dot = dots[(i * VEC + j) & 3];
        dot = fmaf(g[j] * gm[j], n[j], dot);
      }
    }
    const float dot = t.reduce<true, false, false>(RowStats{(dots[0] + dots[1]) + (dots[2] + dots[3]), 0u, 0u}).sq * inv_f;
    T* op = static_cast<T*>(a.gh) + t.row * F;
    FOR_PIECES(i, c) {
      float g[VEC], n[VEC], gm[VEC];
      load_vec(gp + c, g);
      load_q(qp + c, n);
      load_gamma(gamma, c, gm);
#pragma unroll
      for (int j = 0; j < VEC; ++j) g[j] = rstd * (g[j] * gm[j] - n[j] * s * dot);
      if (rp) {
        float r[VEC];
        load_vec(rp + c, r);
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[j] += r[j];
      }
      store_vec(op + c, g);
    }
  }
  t.end();
  if (!a.partial) return;
  // the teams' sums, one after the other, through the ring's memory: every row that was fetched has been waited for
  float* columns = reinterpret_cast<float*>(smem + ring.slots_at);
  for (int w = 0; w < ring.teams; ++w) {
    if (t.team == w) {
      FOR_PIECES(i, c) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) columns[c + j] = w == 0 ? acc[i][j] : columns[c + j] + acc[i][j];
      }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < F; c += CTA) a.partial[static_cast<long long>(blockIdx.x) * F + c] = columns[c];
}
// What the ring does not take: the rows in two passes, the columns by themselves before them (grad_h may be
// grad_out).
template <class T>
__global__ void __launch_bounds__(1024) rmsnorm_bwd_long_rows_kernel(const NormBwdQ8Args a) {
  __shared__ RowStats red[32];
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* gp = static_cast<const T*>(a.go) + row * a.F;
    const T* rp = a.gr ? static_cast<const T*>(a.gr) + row * a.F : nullptr;
    T* op = static_cast<T*>(a.gh) + row * a.F;
    const int8_t* qp = a.hq + row * a.ld;
    const float rstd = a.rstd[row], s = a.hs[row] * rstd;
    RowStats st{0.f, 0u, 0u};
    float g[1], gm[1], r[1] = {0.f};
    for (int c = threadIdx.x; c < a.F; c += blockDim.x) {
      load_vec(gp + c, g);
      load_gamma(a.gamma, c, gm);
      st.sq = fmaf(g[0] * gm[0], static_cast<float>(qp[c]) * s, st.sq);
    }
    const float dot = block_reduce(st, red).sq / static_cast<float>(a.F);
    for (int c = threadIdx.x; c < a.F; c += blockDim.x) {
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
constexpr int RING_BYTES = 216 * 1024;

// The ring's geometry; false where the rows do not fit it (more than 512 * 32 values, fewer than two rows in shared memory,
// pointers off 16-byte boundaries). It depends on the row's length alone, so a row's sums have the same order, and its
// result the same bits, in every batch.
struct RowTensor {
  const void* p;
  long long pitch;   // bytes
  int bytes;
};
bool make_ring(grilly_ctx* ctx, Ring& g, long long rows, int F, const RowTensor* tensors, int count, bool gamma, size_t* smem, unsigned* grid) {
  if (F > CTA * PER_THREAD) return false;
  g = Ring{};
  g.rows = rows;
  g.F = F;
  g.err = ctx->err_dev;
  g.tensors = count;
  g.first_tail = rows;
  for (int i = 0; i < count; ++i) {
    if (reinterpret_cast<uintptr_t>(tensors[i].p) & 15) return false;
    g.src[i] = tensors[i].p;
    g.pitch[i] = tensors[i].pitch;
    g.bytes[i] = tensors[i].bytes;
    g.total[i] = tensors[i].pitch * (rows - 1) + tensors[i].bytes;
    const long long whole = g.total[i] & ~15ll;
    g.first_tail = std::min(g.first_tail, whole < g.bytes[i] ? 0 : (whole - g.bytes[i]) / g.pitch[i] + 1);
    g.at[i] = g.slot;
    g.slot += (tensors[i].bytes + 15) / 16 * 16 + (tensors[i].pitch % 16 ? 16 : 0);
  }
  g.team = 32;
  while (g.team * PER_THREAD < F) g.team *= 2;
  g.teams = CTA / g.team;
  g.gamma_at = GAMMA_AT;
  g.slots_at = GAMMA_AT + (gamma ? (4 * F + 15) / 16 * 16 : 0);
  const int room = RING_BYTES - g.slots_at;
  g.depth = std::min(MAX_DEPTH, room / (g.slot * g.teams));
  // long rows: fewer of them at a time rather than none ahead
  while (g.depth < 2 && g.teams > 1) {
    g.teams /= 2;
    g.depth = std::min(MAX_DEPTH, room / (g.slot * g.teams));
  }
  if (g.depth < 2) return false;
  *grid = static_cast<unsigned>(std::min<long long>(rows, ctx->num_sms));
  const long long per_team = (rows + static_cast<long long>(*grid) * g.teams - 1) / (static_cast<long long>(*grid) * g.teams);
  g.depth = static_cast<int>(std::min<long long>(g.depth, per_team));
  *smem = g.slots_at + std::max(static_cast<size_t>(g.slot) * g.teams * g.depth, sizeof(float) * static_cast<size_t>(F));
  return true;
}
template <class K>
int allow_ring(grilly_ctx* ctx, K kern) {
  const void* key = reinterpret_cast<const void*>(kern);
  if (!ctx->smem_attr_done.count(key)) {
    GB_CUDA_CHECK(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    ctx->smem_attr_done.insert(key);
  }
  return GRILLY_OK;
}
unsigned any_grid(long long rows) { return static_cast<unsigned>(std::min<long long>(rows, 1 << 20)); }

template <class T>
int launch_quantize(grilly_ctx* ctx, const T* x, int8_t* q, float* scale, long long rows, int F, long long ld) {
  constexpr int VEC = 16 / sizeof(T);
  Ring ring;
  size_t smem;
  unsigned grid;
  const RowTensor in[1] = {{x, static_cast<long long>(sizeof(T)) * F, static_cast<int>(sizeof(T)) * F}};
  if (!make_ring(ctx, ring, rows, F, in, 1, false, &smem, &grid)) {
    quantize_long_rows_kernel<<<any_grid(rows), 1024, 0, ctx->stream>>>(x, q, scale, rows, F, ld);
    return GRILLY_OK;
  }
  auto kern = F % VEC == 0 ? quantize_rows_kernel<T, VEC> : quantize_rows_kernel<T, 1>;
  if (int rc = allow_ring(ctx, kern)) return rc;
  kern<<<grid, CTA, smem, ctx->stream>>>(ring, q, scale, ld);
  return GRILLY_OK;
}

template <class T>
void launch_dequantize(grilly_ctx* ctx, const int8_t* q, const float* scale, T* y, long long rows, int F, long long ld) {
  const cudaStream_t st = ctx->stream;
  const long long vectors = rows * (F / 16);
  if (F % 16 == 0 && aligned16({y}) && vectors < (1ll << 31)) {
    const unsigned grid = static_cast<unsigned>(std::min<long long>((vectors + 255) / 256, ctx->num_sms * 32ll));
    dequantize_vec_kernel<T><<<grid, 256, 0, st>>>(q, scale, y, static_cast<uint32_t>(vectors), static_cast<uint32_t>(F / 16), ld);
  } else {
    dequantize_any_kernel<T><<<any_grid((rows + 7) / 8), 256, 0, st>>>(q, scale, y, rows, F, ld);
  }
}

template <class T>
int launch_rmsnorm(grilly_ctx* ctx, const NormQ8Args& a) {
  constexpr int VEC = 16 / sizeof(T);
  Ring ring;
  size_t smem;
  unsigned grid;
  const long long pitch = static_cast<long long>(sizeof(T)) * a.F;
  const RowTensor in[2] = {{a.x, pitch, static_cast<int>(pitch)}, {a.residual, pitch, static_cast<int>(pitch)}};
  if (!aligned16({a.h}) || !make_ring(ctx, ring, a.rows, a.F, in, a.residual ? 2 : 1, a.gamma != nullptr, &smem, &grid)) {
    rmsnorm_q8_long_kernel<T><<<any_grid(a.rows), 1024, 0, ctx->stream>>>(a);
    return GRILLY_OK;
  }
  auto kern = a.F % VEC == 0 ? rmsnorm_q8_kernel<T, VEC> : rmsnorm_q8_kernel<T, 1>;
  if (int rc = allow_ring(ctx, kern)) return rc;
  kern<<<grid, CTA, smem, ctx->stream>>>(ring, a);
  return GRILLY_OK;
}

template <class T>
int launch_rmsnorm_bwd(grilly_ctx* ctx, NormBwdQ8Args& a, float* grad_gamma) {
  constexpr int VEC = 16 / sizeof(T);
  Rows8Scratch scratch(ctx);
  Ring ring;
  size_t smem;
  unsigned grid;
  const long long pitch = static_cast<long long>(sizeof(T)) * a.F;
  const RowTensor in[3] = {{a.hq, a.ld, (a.F + 15) / 16 * 16}, {a.go, pitch, static_cast<int>(pitch)}, {a.gr, pitch, static_cast<int>(pitch)}};
  if (aligned16({a.gh}) && make_ring(ctx, ring, a.rows, a.F, in, a.gr ? 3 : 2, a.gamma != nullptr, &smem, &grid)) {
    auto kern = a.F % VEC == 0 ? rmsnorm_bwd_kernel<T, VEC> : rmsnorm_bwd_kernel<T, 1>;
    if (int rc = allow_ring(ctx, kern)) return rc;
    if (grad_gamma) {
      if (int rc = scratch.take(sizeof(float) * grid * static_cast<size_t>(a.F))) return rc;
      a.partial = static_cast<float*>(scratch.p);
    }
    kern<<<grid, CTA, smem, ctx->stream>>>(ring, a);
    ctx->launches++;
    if (grad_gamma) {
      sum_partials_kernel<<<(a.F + 31) / 32, 512, 0, ctx->stream>>>(a.partial, grad_gamma, static_cast<int>(grid), a.F);
      ctx->launches++;
    }
    GB_CUDA_CHECK(ctx, cudaGetLastError());
    return GRILLY_OK;
  }
  if (grad_gamma) {
    const int blocks = static_cast<int>(std::min<long long>((a.rows + 31) / 32, ctx->num_sms));
    const long long per = (a.rows + blocks - 1) / blocks;
    if (int rc = scratch.take(sizeof(float) * blocks * static_cast<size_t>(a.F))) return rc;
    a.partial = static_cast<float*>(scratch.p);
    rmsnorm_bwd_long_columns_kernel<T><<<blocks, 256, 0, ctx->stream>>>(a, per);
    sum_partials_kernel<<<(a.F + 31) / 32, 512, 0, ctx->stream>>>(a.partial, grad_gamma, blocks, a.F);
    ctx->launches += 2;
  }
  rmsnorm_bwd_long_rows_kernel<T><<<any_grid(a.rows), 1024, 0, ctx->stream>>>(a);
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
    const int rc = bf16 ? launch_quantize(ctx, static_cast<const __nv_bfloat16*>(x), static_cast<int8_t*>(q), scale, rows, features, ld)
                        : launch_quantize(ctx, static_cast<const float*>(x), static_cast<int8_t*>(q), scale, rows, features, ld);
    return rc ? rc : done(ctx, pi);
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
    const int rc = bf16 ? launch_rmsnorm<__nv_bfloat16>(ctx, a) : launch_rmsnorm<float>(ctx, a);
    return rc ? rc : done(ctx, pi);
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
    const double e = bf16 ? 2 : 4, n = static_cast<double>(rows) * features;
    const int pi = prof_begin(ctx, PROF_NORM, 10.0 * n, n * (e * (2 + (grad_residual ? 1 : 0)) + 1) + 8.0 * features + 8.0 * rows);
    const int rc = bf16 ? launch_rmsnorm_bwd<__nv_bfloat16>(ctx, a, grad_gamma) : launch_rmsnorm_bwd<float>(ctx, a, grad_gamma);
    prof_end(ctx, pi);
    return rc;
  });
}

}  // extern "C"
